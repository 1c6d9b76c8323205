"""Cases of the attention and 4-bit product operators: what they compute, in elementary torch operations, and the
calls a program makes of them.

Five kinds of case (``case["kind"]``):

  window   causal attention of a prompt, each query seeing the last ``window`` keys and the first ``sinks`` ones
           (window 0: every key before it); grouped heads; one sequence or a packed ragged batch; a prompt may
           continue a longer key sequence (``prefix`` keys before the first query)
  train    the same, forward and backward
  decode   attention of one new token a sequence over keys and values held in pages
  append   new keys and values written into those pages
  q4       a few vectors times a matrix of 4-bit weights with a scale (and a zero point) per group of columns
"""
import importlib
import math
import pathlib
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _lens(case):
    return [int(t) for t in case["lens"].split(",")]


def listed():
    return [
        # one short sequence of the pruned transformer's shape (512 = 8 heads of 64): latency counts
        dict(name="window-short", kind="window", dtype="fp16", lens="129", prefix=0, heads=8, kv_heads=8, dim=64,
             window=64, sinks=4),
        # a ragged batch packed one after another, each continuing 300 keys, an odd head width, one empty sequence
        # and one of a token
        dict(name="window-ragged", kind="window", dtype="bf16", lens="1,0,77,1023,500,2051,333,64", prefix=300,
             heads=16, kv_heads=4, dim=80, window=256, sinks=4),
        # a long prompt in one piece
        dict(name="window-long", kind="window", dtype="bf16", lens="16384", prefix=0, heads=32, kv_heads=8, dim=128,
             window=2048, sinks=16),
        # a small training step in full precision
        dict(name="train-small", kind="train", dtype="fp32", lens="257", prefix=0, heads=4, kv_heads=2, dim=64,
             window=100, sinks=1),
        # a training step on two long sequences
        dict(name="train-long", kind="train", dtype="bf16", lens="8192,8000", prefix=0, heads=32, kv_heads=8, dim=128,
             window=1024, sinks=4),
        # one user's next token, little behind it: latency counts
        dict(name="decode-one", kind="decode", dtype="fp16", lens="200", heads=8, kv_heads=8, dim=64, page=16,
             window=0, sinks=0),
        # a serving batch of mixed lengths under a window
        dict(name="decode-window", kind="decode", dtype="bf16",
             lens="60001,17,4096,1,933,8191,20000,515,2048,2049,31,7000", heads=32, kv_heads=8, dim=128, page=16,
             window=4096, sinks=64),
        # a full batch of long sequences
        dict(name="decode-large", kind="decode", dtype="bf16",
             lens=",".join(str(16384 - 211 * i) for i in range(32)), heads=64, kv_heads=8, dim=128, page=32,
             window=0, sinks=0),
        # the tokens of one step of a batch
        dict(name="append-step", kind="append", dtype="bf16", lens=",".join(str(100 + 37 * i) for i in range(64)),
             new=1, kv_heads=8, dim=128, page=16),
        # whole prompts
        dict(name="append-prompts", kind="append", dtype="bf16", lens="16384,5001,9000,64,1", new=0, kv_heads=8,
             dim=128, page=64),
        # a projection of the 512-wide transformer, one token, full precision
        dict(name="q4-small", kind="q4", dtype="fp32", tokens=1, rows=512, cols=512, group=32, zeros=False),
        # a wide projection, four tokens, with zero points
        dict(name="q4-large", kind="q4", dtype="fp16", tokens=4, rows=16384, cols=8192, group=128, zeros=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _split(rng, total, parts):
    cuts = sorted(rng.randint(0, total) for _ in range(parts - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    kind = rng.choice(["window", "train", "decode", "append", "q4"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    case = dict(kind=kind, dtype=dtype)
    limits = {c["kind"]: work(c) for c in listed()}         # the last listed case of a kind is its largest
    while True:
        if kind == "q4":
            case.update(tokens=rng.choice([1, 1, 1, 2, 3, 4, 8]), rows=_log(rng, 64, 16384),
                        cols=_log(rng, 64, 8192), group=rng.choice([32, 64, 128, 256]), zeros=rng.random() < 0.5)
        else:
            case.update(kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 80, 96, 128]))
            if kind in ("window", "train"):
                total = _log(rng, 64, 16384 if kind == "window" else 8192)
                lens = _split(rng, total, rng.choice([1, 1, 2, 5]))
                case.update(lens=",".join(map(str, lens)), heads=case["kv_heads"] * rng.choice([1, 2, 4]),
                            prefix=rng.choice([0, 0, rng.randint(1, 2000)]) if kind == "window" else 0,
                            window=rng.choice([0, _log(rng, 16, 4096), _log(rng, 16, 4096)]),
                            sinks=rng.choice([0, 1, 4, 64]))
                if dtype == "fp32" and work(case)["flops"] > 2e10:       # full precision stands for small models
                    continue
            elif kind == "decode":
                batch = _log(rng, 1, 32)
                lens = [_log(rng, 1, 32768) for _ in range(batch)]
                case.update(lens=",".join(map(str, lens)), heads=case["kv_heads"] * rng.choice([1, 2, 4, 8]),
                            page=rng.choice([8, 16, 32, 64, 256]), window=rng.choice([0, 0, _log(rng, 64, 8192)]),
                            sinks=rng.choice([0, 4, 64]))
            else:
                batch = _log(rng, 1, 64)
                new = rng.choice([0, 1, 1, 5])
                lens = [max(new, _log(rng, 1, 4096)) for _ in range(batch)]
                case.update(lens=",".join(map(str, lens)), new=new, page=rng.choice([8, 16, 32, 64, 256]))
        w = work(case)
        if w["bytes"] <= limits[kind]["bytes"] * 1.0001 and w["flops"] <= limits[kind]["flops"] * 1.0001:
            if kind != "append" or sum(_lens(case)) <= 32768:            # the pages are part of what comes back
                return case


def _ramp(n, top):
    """Sum of min(i, top) for i in 1..n."""
    t = min(n, top)
    return t * (t + 1) // 2 + (n - t) * top if n > 0 else 0


def _visible(n_q, n_k, window, sinks):
    """Visible (query, key) pairs of one head: query i sits at position i + n_k - n_q."""
    def upto(n):                                    # pairs of the queries at positions 0..n-1
        return _ramp(n, window) + _ramp(n - window, sinks) if window else _ramp(n, n)
    return upto(n_k) - upto(n_k - n_q)


def work(case):
    kind, b = case["kind"], BYTES[case["dtype"]]
    if kind == "q4":
        n, k, t = case["rows"], case["cols"], case["tokens"]
        groups = -(-k // case["group"])
        return {"bytes": n * ((k + 1) // 2) + n * groups * (b + (1 if case["zeros"] else 0)) + t * (n + k) * b,
                "flops": 2 * n * k * t}
    lens, d, hkv = _lens(case), case["dim"], case["kv_heads"]
    if kind == "append":
        new = sum(n if case["new"] == 0 else case["new"] for n in lens)
        return {"bytes": 2 * 2 * new * hkv * d * b + 8 * len(lens), "flops": 0}
    h = case["heads"]
    if kind == "decode":
        keys = sum(_visible(1, n, case["window"], case["sinks"]) for n in lens)
        return {"bytes": 2 * keys * hkv * d * b + 2 * len(lens) * h * d * b + 4 * len(lens) * h,
                "flops": 4 * keys * h * d}
    nq, nk = sum(lens), sum(n + case["prefix"] if n else 0 for n in lens)
    pairs = h * sum(_visible(n, n + case["prefix"], case["window"], case["sinks"]) for n in lens if n)
    qo, kv = nq * h * d * b, nk * hkv * d * b
    fwd = {"bytes": 2 * qo + 2 * kv + 4 * nq * h, "flops": 4 * pairs * d}
    if kind == "window":
        return fwd
    # q, k, v and the output's gradient in; the output and three gradients out; two products forward, five backward
    return {"bytes": 4 * qo + 4 * kv + 4 * nq * h, "flops": 14 * pairs * d}


def prepare(case, seed):
    st = _inputs(case, seed)
    if own and case["kind"] == "q4":
        # the weights are laid out once, when a program loads them
        st["format"] = _package("q4").Q4Format(st["packed"], st["scales"], st["z"], cols=case["cols"],
                                               group=case["group"])
    return st


def _package(module):
    root = str(pathlib.Path(__file__).resolve().parents[1] / "spmm-research_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    return importlib.import_module("spmm_amd." + module)


def _inputs(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    st = dict(case)
    if case["kind"] == "q4":
        n, k = case["rows"], case["cols"]
        groups = -(-k // case["group"])
        st["packed"] = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device=dev, dtype=torch.uint8)
        st["scales"] = (0.01 * (0.5 + torch.rand(n, groups, generator=g, device=dev))).to(dt)
        st["z"] = (torch.randint(5, 12, (n, groups), generator=g, device=dev, dtype=torch.uint8)
                   if case["zeros"] else None)
        st["x"] = randn(case["tokens"], k)
        return st
    lens, d, hkv = _lens(case), case["dim"], case["kv_heads"]
    st["host_lens"] = lens
    if case["kind"] in ("window", "train"):
        # queries, keys and values as one projection leaves them: views of one buffer
        h, nq = case["heads"], sum(lens)
        klens = [n + case["prefix"] if n else 0 for n in lens]
        st["k_lens"] = klens
        if case["prefix"]:
            st["q"] = randn(nq, h, d)
            kv = randn(sum(klens), 2 * hkv, d)
            st["k"], st["v"] = kv[:, :hkv], kv[:, hkv:]
        else:
            qkv = randn(nq, h + 2 * hkv, d)
            st["q"], st["k"], st["v"] = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
        st["cu_q"] = _offsets(lens, dev)
        st["cu_k"] = _offsets(klens, dev)
        if case["kind"] == "train":
            st["dout"] = randn(nq, h, d)
        return st
    # pages in an order of their own, a few more than the sequences use
    page = case["page"]
    used = [-(-n // page) for n in lens]
    pool = sum(used) + 5
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(used)), -1, device=dev, dtype=torch.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    st["table"] = table
    st["lengths"] = torch.tensor(lens, device=dev, dtype=torch.int32)
    st["max_length"] = max(lens)
    st["k_pages"], st["v_pages"] = (torch.empty(pool, page, hkv, d, device=dev, dtype=dt) for _ in range(2))
    for pages in (st["k_pages"], st["v_pages"]):
        pages.normal_(generator=g)
    if case["kind"] == "decode":
        st["q"] = randn(len(lens), case["heads"], d)
    else:
        new = [n if case["new"] == 0 else case["new"] for n in lens]
        st["new_lens"] = new
        st["k"], st["v"] = randn(sum(new), hkv, d), randn(sum(new), hkv, d)
        st["cu"] = _offsets(new, dev) if case["new"] != 1 else None
    return st


def _offsets(lens, dev):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, device=dev, dtype=torch.int32)


def run(state):
    return (_run_own if own else _run_plain)(state)


# ------------------------------------------------------------------------------------- the framework's calls
def _run_own(st):
    kind = st["kind"]
    if kind == "q4":
        return st["format"].matvec(st["x"])
    A = _package("attention")
    if kind == "append":
        A.cache_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["lengths"], cu=st["cu"])
        return st["k_pages"], st["v_pages"]
    mask = dict(window=st["window"], sinks=st["sinks"])
    if kind == "decode":
        return A.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"],
                                 max_length=st["max_length"], **mask)
    out, lse = A.window_attention(st["q"], st["k"], st["v"], cu_q=st["cu_q"], cu_k=st["cu_k"], **mask)
    if kind == "window":
        return out, lse
    dq, dk, dv = A.window_attention_backward(st["dout"], st["q"], st["k"], st["v"], out, lse, cu_q=st["cu_q"],
                                             cu_k=st["cu_k"], **mask)
    return out, lse, dq, dk, dv


# ------------------------------------------------------------------------------------- plain forms
def _run_plain(st):
    return {"q4": _plain_q4, "append": _plain_append, "decode": _plain_decode, "window": _plain_window,
            "train": _plain_train}[st["kind"]](st)


def _plain_q4(st):
    n, k, group = st["rows"], st["cols"], st["group"]
    q = torch.stack((st["packed"] & 15, st["packed"] >> 4), dim=2).reshape(n, -1)[:, :k].float()
    col = torch.arange(k, device=q.device) // group
    zero = st["z"].float()[:, col] if st["z"] is not None else 8.0
    w = (q - zero) * st["scales"].float()[:, col]
    return (st["x"].float() @ w.t()).to(st["x"].dtype)


def _plain_append(st):
    kp, vp, page = st["k_pages"], st["v_pages"], st["page"]
    cu = st["cu"].long() if st["cu"] is not None else torch.arange(len(st["lengths"]) + 1, device=kp.device)
    row = torch.arange(st["k"].shape[0], device=kp.device)
    seq = torch.searchsorted(cu, row, right=True) - 1
    pos = st["lengths"].long()[seq] - cu[seq + 1] + row
    pg = st["table"].long()[seq, pos // page]
    kp[pg, pos % page] = st["k"]
    vp[pg, pos % page] = st["v"]
    return kp, vp


def _softmax_parts(s):
    """Weights and log-sum of the rows of s (masked places at -inf; no row is empty here)."""
    m = s.amax(-1, keepdim=True)
    p = (s - m).exp_()
    total = p.sum(-1, keepdim=True)
    return p / total, (m + total.log()).squeeze(-1)


def _plain_decode(st):
    q, d, page = st["q"], st["dim"], st["page"]
    hkv, h = st["kv_heads"], st["heads"]
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], device=q.device, dtype=torch.float32)
    for i, n in enumerate(st["host_lens"]):
        pos = torch.arange(n, device=q.device)
        if st["window"]:
            pos = pos[(pos >= n - st["window"]) | (pos < st["sinks"])]
        pg = st["table"][i].long()[pos // page]
        k = st["k_pages"][pg, pos % page].float().permute(1, 2, 0).contiguous()      # [hkv, d, keys]
        v = st["v_pages"][pg, pos % page].float().transpose(0, 1).contiguous()       # [hkv, keys, d]
        p, z = _softmax_parts(q[i].float().reshape(hkv, h // hkv, d) @ k * d ** -0.5)
        out[i] = (p @ v).reshape(h, d).to(q.dtype)
        lse[i] = z.reshape(h)
    return out, lse


def _blocks(st, rows=512):
    """Blocks of queries with the keys that some query of the block sees: (query slice, key indices, mask)."""
    q0 = k0 = 0
    dev = st["q"].device
    for n, nk in zip(st["host_lens"], st["k_lens"]):
        for a in range(0, n, rows):
            b = min(n, a + rows)
            shift = nk - n
            lo = max(0, a + shift - st["window"] + 1) if st["window"] else 0
            keys = torch.arange(lo, b + shift, device=dev)
            if min(st["sinks"], lo):
                keys = torch.cat((torch.arange(min(st["sinks"], lo), device=dev), keys))
            p = torch.arange(a + shift, b + shift, device=dev)[:, None]
            seen = keys <= p
            if st["window"]:
                seen &= (p - keys < st["window"]) | (keys < st["sinks"])
            yield slice(q0 + a, q0 + b), k0 + keys, seen
        q0 += n
        k0 += nk


def _grouped(x, hkv):
    """[rows, heads, d] -> [hkv, heads / hkv * rows, d] in 32 bits."""
    r, h, d = x.shape
    return x.float().reshape(r, hkv, h // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)


def _ungrouped(x, r, h):
    hkv, d = x.shape[0], x.shape[-1]
    return x.reshape(hkv, h // hkv, r, d).permute(2, 0, 1, 3).reshape(r, h, d)


def _plain_window(st, train=False):
    q, k, v, hkv, h, d = st["q"], st["k"], st["v"], st["kv_heads"], st["heads"], st["dim"]
    scale = d ** -0.5
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    lse = torch.empty(q.shape[:2], device=q.device, dtype=torch.float32)
    if train:
        dq = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        dk, dv = (torch.zeros(k.shape, device=q.device, dtype=torch.float32) for _ in range(2))
    for rows, keys, seen in _blocks(st):
        r = rows.stop - rows.start
        qb = _grouped(q[rows], hkv)
        kb = k[keys].float().transpose(0, 1).contiguous()
        vb = v[keys].float().transpose(0, 1).contiguous()
        s = qb @ kb.transpose(1, 2).contiguous() * scale
        s = s.reshape(hkv, h // hkv, r, -1).masked_fill_(~seen, float("-inf")).reshape(hkv, -1, len(keys))
        p, z = _softmax_parts(s)
        o = p @ vb
        out[rows] = _ungrouped(o, r, h).to(q.dtype)
        lse[rows] = _ungrouped(z[..., None], r, h)[..., 0]
        if train:
            do = _grouped(st["dout"][rows], hkv)
            ds = p * (do @ vb.transpose(1, 2).contiguous() - (do * o).sum(-1, keepdim=True))
            dq[rows] = _ungrouped(ds @ kb * scale, r, h).to(q.dtype)
            dk.index_add_(0, keys, (ds.transpose(1, 2).contiguous() @ qb * scale).transpose(0, 1))
            dv.index_add_(0, keys, (p.transpose(1, 2).contiguous() @ do).transpose(0, 1))
    if train:
        return out, lse, dq, dk.to(k.dtype), dv.to(v.dtype)
    return out, lse


def _plain_train(st):
    return _plain_window(st, train=True)


# ------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    st = _inputs(case, seed)
    kind = case["kind"]
    if kind == "append":                         # rows are copied, not computed: by flat slots
        pools = []
        for pages, rows in ((st["k_pages"], st["k"]), (st["v_pages"], st["v"])):
            flat, at = pages.double().flatten(0, 1), 0
            for i, new in enumerate(st["new_lens"]):
                for j in range(0, new, case["page"]):
                    pos = torch.arange(j, min(new, j + case["page"]), device="cuda") + st["host_lens"][i] - new
                    slot = st["table"][i].long()[pos // case["page"]] * case["page"] + pos % case["page"]
                    flat[slot] = rows[at + j:at + j + len(pos)].double()
                at += new
            pools.append(flat.reshape(pages.shape))
        return tuple(pools)
    if kind == "q4":
        y = torch.zeros(case["tokens"], case["rows"], device="cuda", dtype=torch.float64)
        x = st["x"].double()
        for g, c0 in enumerate(range(0, case["cols"], case["group"])):
            c = torch.arange(c0, min(case["cols"], c0 + case["group"]), device="cuda")
            byte = st["packed"][:, c // 2].int()
            w = (byte >> (4 * (c % 2)).int()) % 16
            w = w.double() - (st["z"][:, g:g + 1].double() if st["z"] is not None else 8.0)
            y += st["scales"][:, g].double() * torch.matmul(x[:, c], w.t().contiguous())
        return y
    d, h, hkv = case["dim"], case["heads"], case["kv_heads"]
    group, scale, w, sinks = h // hkv, 1.0 / math.sqrt(case["dim"]), case["window"], case["sinks"]
    if kind == "decode":
        out = torch.empty(len(st["host_lens"]), h, d, device="cuda", dtype=torch.float64)
        lse = torch.empty(out.shape[:2], device="cuda", dtype=torch.float64)
        for i, n in enumerate(st["host_lens"]):
            used = st["table"][i, :-(-n // case["page"])].long()
            for kh in range(hkv):
                k = st["k_pages"][used, :, kh].reshape(-1, d)[:n].double()
                v = st["v_pages"][used, :, kh].reshape(-1, d)[:n].double()
                s = torch.matmul(st["q"][i, kh * group:(kh + 1) * group].double(), k.t().contiguous()) * scale
                if w and n > w:
                    s[:, min(sinks, n - w):n - w] = float("-inf")
                z = torch.logsumexp(s, dim=1)
                out[i, kh * group:(kh + 1) * group] = torch.matmul(torch.exp(s - z[:, None]), v)
                lse[i, kh * group:(kh + 1) * group] = z
        return out, lse
    train = kind == "train"
    q, k, v = st["q"], st["k"], st["v"]
    out = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    lse = torch.zeros(q.shape[:2], device="cuda", dtype=torch.float64)
    dq, dk, dv = (torch.zeros(t.shape, device="cuda", dtype=torch.float64) for t in (q, k, v)) if train else (None,) * 3
    q0 = k0 = 0
    for n, nk in zip(st["host_lens"], st["k_lens"]):
        for head in range(h):
            kh = head // group
            ks, vs = k[k0:k0 + nk, kh].double(), v[k0:k0 + nk, kh].double()
            for a in range(0, n, 1024):
                rows = torch.arange(a, min(n, a + 1024), device="cuda")
                p = rows + nk - n
                first = max(0, a + nk - n - w + 1) if w else 0
                cols = torch.arange(nk, device="cuda")
                cols = cols[((cols >= first) | (cols < sinks)) & (cols <= p[-1])]
                hidden = cols[None, :] > p[:, None]
                if w:
                    hidden = hidden | ((cols[None, :] <= p[:, None] - w) & (cols[None, :] >= sinks))
                qs = q[q0 + rows, head].double()
                kc, vc = ks[cols], vs[cols]
                s = torch.where(hidden, -math.inf, torch.matmul(qs, kc.t().contiguous()) * scale)
                z = torch.logsumexp(s, dim=1)
                weight = torch.exp(s - z[:, None])
                o = torch.matmul(weight, vc)
                out[q0 + rows, head], lse[q0 + rows, head] = o, z
                if train:
                    do = st["dout"][q0 + rows, head].double()
                    dw = torch.matmul(do, vc.t().contiguous())
                    ds = weight * (dw - (weight * dw).sum(1, keepdim=True)) * scale
                    dq[q0 + rows, head] = torch.matmul(ds, kc)
                    dk[k0 + cols, kh] += torch.matmul(ds.t().contiguous(), qs)
                    dv[k0 + cols, kh] += torch.matmul(weight.t().contiguous(), do)
        q0 += n
        k0 += nk
    return (out, lse, dq, dk, dv) if train else (out, lse)
