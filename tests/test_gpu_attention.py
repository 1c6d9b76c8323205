"""Window attention, its gradients, attention over pages and the append, on the GPU against float64 (attention_oracle)."""
import itertools
import math

import pytest
import torch

import attention_oracle as O

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TYPES = [BF16, F16, F32]


@pytest.fixture(scope="module")
def A():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import attention
    return attention


def rnd(seed, *shape, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# (queries, keys, heads, key heads, width, window, sinks)
WINDOW = [
    (1, 1, 1, 1, 1, 0, 0), (1, 1, 2, 1, 64, 1, 0), (5, 5, 3, 3, 8, 2, 1), (33, 33, 4, 2, 17, 7, 3),
    (128, 128, 2, 1, 64, 0, 0), (129, 129, 8, 8, 64, 64, 4), (200, 300, 4, 1, 80, 50, 4), (64, 700, 4, 2, 96, 130, 70),
    (257, 257, 4, 2, 128, 100, 1), (131, 131, 2, 2, 100, 1, 0), (300, 300, 2, 1, 128, 64, 130), (90, 40, 2, 1, 64, 16, 4),
    (3, 0, 2, 1, 64, 4, 1), (260, 260, 6, 2, 33, 0, 5), (400, 401, 2, 1, 72, 400, 0), (1, 513, 4, 4, 128, 200, 8),
    (150, 150, 16, 1, 64, 33, 32), (321, 321, 2, 1, 128, 320, 2),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", WINDOW, ids=str)
def test_window_and_gradients(A, case, dtype):
    nq, nk, h, hk, d, window, sinks = case
    q, k, v = rnd(1, nq, h, d, dtype=dtype), rnd(2, nk, hk, d, dtype=dtype), rnd(3, nk, hk, d, dtype=dtype)
    do = rnd(4, nq, h, d, dtype=dtype)
    out, lse = A.window_attention(q[None], k[None], v[None], window, sinks)
    r = O.attention(q, k, v, window, sinks)
    O.check("out", out[0], r["out"], r["tol_out"])
    O.check("lse", lse[0], r["lse"], r["tol_lse"])
    got = A.window_attention_backward(do[None], q[None], k[None], v[None], out, lse, window, sinks)
    g = O.gradients(r, do)
    for name, x in zip(("dq", "dk", "dv"), got):
        O.check(name, x[0], g[name], g["tol_" + name])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0, 4.0])
def test_scales(A, dtype, scale):
    q, k, v = (rnd(i, 70, 2, 40, dtype=dtype) for i in (1, 2, 3))
    do = rnd(4, 70, 2, 40, dtype=dtype)
    out, lse = A.window_attention(q[None], k[None], v[None], 20, 3, scale)
    r = O.attention(q, k, v, 20, 3, scale)
    O.check("out", out[0], r["out"], r["tol_out"])
    O.check("lse", lse[0], r["lse"], r["tol_lse"])
    got = A.window_attention_backward(do[None], q[None], k[None], v[None], out, lse, 20, 3, scale)
    g = O.gradients(r, do)
    for name, x in zip(("dq", "dk", "dv"), got):
        O.check(name, x[0], g[name], g["tol_" + name])


def test_gradients_against_differences(A):
    """float32: the gradient along a direction against a central difference of sum(out * w) in float64."""
    nq, nk, h, hk, d, window, sinks = 20, 30, 4, 2, 24, 9, 2
    q, k, v, w = rnd(1, nq, h, d), rnd(2, nk, hk, d), rnd(3, nk, hk, d), rnd(4, nq, h, d)
    out, lse = A.window_attention(q[None], k[None], v[None], window, sinks)
    grads = [x[0].cpu().double() for x in A.window_attention_backward(w[None], q[None], k[None], v[None], out, lse, window, sinks)]
    x0 = [t.cpu().double() for t in (q, k, v)]
    f = lambda xs: (O.attention(*xs, window, sinks)["out"] * w.cpu().double()).sum()
    for i in range(3):
        for seed in range(3):
            step = torch.randn(x0[i].shape, generator=torch.Generator().manual_seed(50 + seed)).double()
            e = 1e-5
            plus, minus = list(x0), list(x0)
            plus[i], minus[i] = x0[i] + e * step, x0[i] - e * step
            slope = (f(plus) - f(minus)) / (2 * e)
            r = O.attention(q, k, v, window, sinks)
            tol = (O.gradients(r, w)[("tol_dq", "tol_dk", "tol_dv")[i]] * step.abs()).sum() + 1e-7 * abs(slope) + 1e-7
            assert abs((grads[i] * step).sum() - slope) <= tol


LENS = [([1, 0, 77, 130, 5], [1, 0, 77, 130, 5]), ([0, 0, 3], [4, 0, 9]), ([128, 256], [128, 300]), ([200], [200]),
        ([1] * 70, [3] * 70), ([5, 0, 129], [2, 6, 129])]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lens", LENS, ids=lambda x: str(x)[:40])
def test_packed(A, lens, dtype):
    """A ragged batch in one buffer: every sequence as if alone; rows behind the last zeroed, or left if given."""
    lq, lk = lens
    h, hk, d, window, sinks, rest = 4, 2, 48, 40, 2, 150
    q, k, v = rnd(1, sum(lq) + rest, h, d, dtype=dtype), *(rnd(i, sum(lk) + rest, hk, d, dtype=dtype) for i in (2, 3))
    do = rnd(4, *q.shape, dtype=dtype)
    cu = [torch.tensor([0] + list(itertools.accumulate(x)), dtype=torch.int32).cuda() for x in (lq, lk)]
    q[sum(lq):] = k[sum(lk):] = v[sum(lk):] = do[sum(lq):] = float("nan")
    args = dict(window=window, sinks=sinks, cu_q=cu[0], cu_k=cu[1])
    out, lse = A.window_attention(q, k, v, **args)
    grads = A.window_attention_backward(do, q, k, v, out, lse, **args)
    a = b = 0
    for nq, nk in zip(lq, lk):
        r = O.attention(q[a:a + nq], k[b:b + nk], v[b:b + nk], window, sinks)
        O.check("out", out[a:a + nq], r["out"], r["tol_out"])
        O.check("lse", lse[a:a + nq], r["lse"], r["tol_lse"])
        g = O.gradients(r, do[a:a + nq])
        for name, x, s in (("dq", grads[0], slice(a, a + nq)), ("dk", grads[1], slice(b, b + nk)), ("dv", grads[2], slice(b, b + nk))):
            O.check(name, x[s], g[name], g["tol_" + name])
        a, b = a + nq, b + nk
    assert (out[a:] == 0).all() and (lse[a:] == -math.inf).all()
    assert (grads[0][a:] == 0).all() and (grads[1][b:] == 0).all() and (grads[2][b:] == 0).all()
    out2, lse2 = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
    g2 = [torch.full_like(x, 7.0) for x in grads]
    A.window_attention(q, k, v, **args, out=out2, lse=lse2)
    A.window_attention_backward(do, q, k, v, out2, lse2, **args, dq=g2[0], dk=g2[1], dv=g2[2])
    assert torch.equal(out2[:a], out[:a]) and (out2[a:] == 7).all() and (lse2[a:] == 7).all()
    for x, y, n in zip(g2, grads, (a, b, b)):
        assert torch.equal(x[:n], y[:n]) and (x[n:] == 7).all()


def test_packed_without_sequences(A):
    q, cu = rnd(1, 9, 2, 16), torch.zeros(1, dtype=torch.int32).cuda()
    out, lse = A.window_attention(q, q, q, cu_q=cu)
    assert (out == 0).all() and (lse == -math.inf).all()
    for g in A.window_attention_backward(q, q, q, q, out, lse, cu_q=cu):
        assert (g == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_strides(A, dtype, shift):
    """Heads before rows, one buffer for q, k and v, and addresses off every vector's alignment."""
    b, n, h, hk, d = 2, 100, 4, 2, 40
    whole = rnd(1, b, n, (h + 2 * hk) * d + 8, dtype=dtype).flatten()
    whole = torch.cat((whole, whole[:16]))[shift:shift + b * n * ((h + 2 * hk) * d + 8)].reshape(b, n, -1)[..., :(h + 2 * hk) * d]
    q, k, v = whole.unflatten(-1, (h + 2 * hk, d)).split((h, hk, hk), 2)
    do = rnd(2, b, h, n, d, dtype=dtype).transpose(1, 2)
    out = torch.zeros(b, h, n, d + shift, dtype=dtype).cuda()[..., :d].transpose(1, 2)
    out2, lse = A.window_attention(q, k, v, 30, 2, out=out)
    assert out2 is out
    gq, gk, gv = (torch.zeros(n, t.shape[2], b, d + shift, dtype=dtype).cuda()[..., shift:].permute(2, 0, 1, 3) for t in (q, k, v))
    A.window_attention_backward(do, q, k, v, out, lse, 30, 2, dq=gq, dk=gk, dv=gv)
    for i in range(b):
        r = O.attention(q[i], k[i], v[i], 30, 2)
        O.check("out", out[i], r["out"], r["tol_out"])
        g = O.gradients(r, do[i])
        for name, x in (("dq", gq), ("dk", gk), ("dv", gv)):
            O.check(name, x[i], g[name], g["tol_" + name])


def test_broadcast_operands(A):
    """Keys and values of one head shown as several (stride 0), and one sequence as two."""
    q, k, v, do = rnd(1, 2, 60, 4, 32), rnd(2, 1, 60, 1, 32), rnd(3, 1, 60, 1, 32), rnd(4, 2, 60, 4, 32)
    ke, ve = k.expand(2, 60, 2, 32), v.expand(2, 60, 2, 32)
    out, lse = A.window_attention(q, ke, ve, 11, 1)
    dq, dk, dv = A.window_attention_backward(do, q, ke, ve, out, lse, 11, 1)
    ref = A.window_attention(q, ke.contiguous(), ve.contiguous(), 11, 1)
    assert torch.equal(out, ref[0]) and torch.equal(lse, ref[1])
    for i in range(2):
        g = O.gradients(O.attention(q[i], ke[i], ve[i], 11, 1), do[i])
        for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):
            O.check(name, x[i], g[name], g["tol_" + name])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", [0, 5, 70, 129])
def test_masked_places_do_not_leak(A, dtype, value, where):
    """A key, value, query or gradient row that is not finite changes nothing for those that do not see it."""
    n, h, hk, d, window, sinks = 200, 2, 1, 64, 40, 2
    base = [rnd(i, n, h if i in (1, 4) else hk, d, dtype=dtype) for i in (1, 2, 3, 4)]
    seen = O.visible(n, n, window, sinks)
    rows = ~seen[:, where]                               # queries that do not see the key
    keys = ~seen[where]                                  # keys that the query does not see
    run = lambda q, k, v, do: (lambda o, l: (o, l) + A.window_attention_backward(
        do[None], q[None], k[None], v[None], o, l, window, sinks))(*A.window_attention(q[None], k[None], v[None], window, sinks))
    ref = [x[0] for x in run(*base)]
    for i in range(4):
        x = [t.clone() for t in base]
        x[i][where, :, 3] = value
        got = [y[0] for y in run(*x)]
        if i in (1, 2):                                  # a key or a value
            assert torch.equal(got[0][rows], ref[0][rows]) and torch.equal(got[1][rows], ref[1][rows])
            assert torch.equal(got[2][rows], ref[2][rows])
            if i == 2:                                   # seen: as the value says
                s = got[0][~rows][..., 3].float()
                assert (s.isnan() if math.isnan(value) else s == value).all()
        else:                                            # a query or its gradient
            other = torch.arange(n) != where
            assert torch.equal(got[0][other], ref[0][other]) and torch.equal(got[2][other], ref[2][other])
            assert torch.equal(got[3][keys], ref[3][keys]) and torch.equal(got[4][keys], ref[4][keys])
            if i == 3:
                assert not torch.isfinite(got[4][~keys][..., 3]).any()


def test_keys_no_query_sees_may_be_anything(A):
    """Keys before the first query's window, past the first keys that stay."""
    q, k, v = rnd(1, 1, 40, 2, 64), rnd(2, 1, 400, 2, 64), rnd(3, 1, 400, 2, 64)
    ref = A.window_attention(q, k, v, 50, 4)
    k[:, 4:311] = v[:, 4:311] = float("nan")
    got = A.window_attention(q, k, v, 50, 4)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_large_scores(A):
    """Scores far beyond the exponential's range, of both signs."""
    q, k, v = rnd(1, 90, 2, 64, scale=40.0), rnd(2, 90, 2, 64, scale=40.0), rnd(3, 90, 2, 64)
    out, lse = A.window_attention(q[None], k[None], v[None], 33, 1)
    r = O.attention(q, k, v, 33, 1)
    O.check("out", out[0], r["out"], r["tol_out"])
    O.check("lse", lse[0], r["lse"], r["tol_lse"])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_repeated_runs_agree(A, dtype):
    q, k, v, do = (rnd(i, 2, 500, 4, 64, dtype=dtype) for i in (1, 2, 3, 4))
    runs = []
    for _ in range(3):
        out, lse = A.window_attention(q, k, v, 100, 4)
        runs.append((out, lse) + A.window_attention_backward(do, q, k, v, out, lse, 100, 4))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


# ------------------------------------------------------------------------------------------------ pages
def make_cache(lens, page, hk, d, dtype, seed=9, extra=3, order="page"):
    """Pages in a shuffled order, unused rows NaN; the sequences' keys and values beside them."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lens]
    total = sum(used) + extra
    perm = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lens), max(used + [1])), -7, dtype=torch.int32)
    shape = {"page": (total, page, hk, d), "head": (total, hk, page, d)}[order]
    kp, vp = (torch.full(shape, float("nan"), dtype=dtype) for _ in range(2))
    view = (lambda t: t) if order == "page" else (lambda t: t.transpose(1, 2))
    ks, vs, at = [], [], 0
    for i, n in enumerate(lens):
        k, v = (torch.randn(n, hk, d, generator=g).to(dtype) for _ in range(2))
        for j in range(used[i]):
            p = perm[at]
            at += 1
            table[i, j] = p
            rows = k[j * page:(j + 1) * page]
            view(kp)[p, :len(rows)], view(vp)[p, :len(rows)] = rows, v[j * page:(j + 1) * page]
        ks.append(k)
        vs.append(v)
    return view(kp.cuda()), view(vp.cuda()), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), ks, vs


def check_paged(A, q, ks, vs, out, lse, window, sinks):
    for i, (k, v) in enumerate(zip(ks, vs)):
        if len(k) == 0:
            assert (out[i] == 0).all() and (lse[i] == -math.inf).all()
            continue
        r = O.attention(q[i:i + 1], k, v, window, sinks, rounded_weights=False)
        O.check(f"out of {len(k)}", out[i:i + 1], r["out"], r["tol_out"])
        O.check(f"lse of {len(k)}", lse[i:i + 1], r["lse"], r["tol_lse"])


# (lengths, heads, key heads, width, page, window, sinks)
PAGED = [
    ([1], 1, 1, 1, 1, 0, 0), ([1, 0, 17], 2, 1, 64, 16, 0, 0), ([200], 8, 8, 64, 16, 0, 0), ([33, 700, 64, 5], 8, 2, 128, 16, 0, 0),
    ([500, 499, 3], 16, 1, 128, 32, 100, 4), ([1000], 4, 2, 80, 8, 64, 70), ([3000, 10], 8, 1, 96, 256, 0, 0),
    ([129, 128, 127], 20, 1, 64, 3, 50, 7), ([2049], 34, 2, 40, 16, 1, 0), ([777, 300], 6, 3, 33, 7, 300, 1),
    ([0, 0], 4, 2, 64, 16, 8, 2), ([5000], 8, 8, 128, 64, 4096, 64), ([90], 4, 4, 128, 16, 89, 0), ([90], 4, 4, 100, 16, 90, 0),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", PAGED, ids=lambda c: str(c)[:60])
def test_paged(A, case, dtype):
    lens, h, hk, d, page, window, sinks = case
    kp, vp, table, lengths, ks, vs = make_cache(lens, page, hk, d, dtype)
    q = rnd(5, len(lens), h, d, dtype=dtype)
    for longest in (None, max(lens)):
        out, lse = A.paged_attention(q, kp, vp, table, lengths, window, sinks, max_length=longest)
        check_paged(A, q, ks, vs, out, lse, window, sinks)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_paged_strides(A, dtype):
    """Heads before rows in a page, a slice of the heads, a table that is a slice, outputs in place."""
    kp, vp, table, lengths, ks, vs = make_cache([300, 41], 16, 4, 64, dtype, order="head")
    wide = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32).cuda()
    wide[:, 2:2 + table.shape[1]] = table
    q = rnd(5, 3, 2, 64, dtype=dtype).transpose(0, 1)[:, :2]
    out = torch.zeros(2, 2, 67, dtype=dtype).cuda()[..., 3:]
    A.paged_attention(q, kp[:, :, 1:3], vp[:, :, 1:3], wide[:, 2:2 + table.shape[1]], lengths, 60, 4, out=out)
    for i in range(2):
        r = O.attention(q[i:i + 1], ks[i][:, 1:3], vs[i][:, 1:3], 60, 4, rounded_weights=False)
        O.check("out", out[i:i + 1], r["out"], r["tol_out"])
    # off every vector's alignment
    flat = torch.zeros(kp.numel() + 1, dtype=dtype).cuda()
    kq = flat[1:].view(kp.shape[0], kp.shape[1], kp.shape[2], kp.shape[3]).copy_(kp)
    o2, l2 = A.paged_attention(q, kq[:, :, 1:3], vp[:, :, 1:3], table, lengths, 60, 4)
    assert torch.equal(o2, out)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_paged_bad_pages_and_lengths(A, dtype):
    """A page that is not there or a length that cannot be: NaN for that sequence alone, if it is seen at all."""
    lens = [300, 300, 300, 300, 300, 300]
    kp, vp, table, lengths, ks, vs = make_cache(lens, 16, 2, 64, dtype)
    q = rnd(5, 6, 4, 64, dtype=dtype)
    ref, rl = A.paged_attention(q, kp, vp, table, lengths, 100, 4)
    table[1, 15], table[2, 15], table[3, 5] = kp.shape[0], -1, 2 ** 31 - 1     # the last is outside what is seen
    lengths[4], lengths[5] = -1, 16 * table.shape[1] + 1
    out, lse = A.paged_attention(q, kp, vp, table, lengths, 100, 4)
    for i in (0, 3):
        assert torch.equal(out[i], ref[i]) and torch.equal(lse[i], rl[i])
    for i in (1, 2, 4, 5):
        assert out[i].isnan().all() and lse[i].isnan().all()
    lengths[:] = 300
    out, lse = A.paged_attention(q, kp, vp, table, lengths, 100, 4, max_length=299)
    assert out.isnan().all() and lse.isnan().all()


def test_paged_far_offsets(A):
    """Pages past 2^31 elements and 2^32 bytes from the first."""
    page, hk, d = 64, 8, 128
    n = 2 ** 31 // (page * hk * d) + 70
    kp, vp = (torch.zeros(n, page, hk, d, dtype=BF16, device="cuda") for _ in range(2))
    lens = [200, 1]
    table = torch.tensor([[n - 1, 3, n - 2, n - 40], [n - 5, 0, 0, 0]], dtype=torch.int32).cuda()
    lengths = torch.tensor(lens, dtype=torch.int32).cuda()
    k, v = rnd(1, 201, hk, d, dtype=BF16), rnd(2, 201, hk, d, dtype=BF16)
    cu = torch.tensor([0, 200, 201], dtype=torch.int32).cuda()
    A.cache_append(k, v, kp, vp, table, lengths, cu)
    q = rnd(3, 2, 16, d, dtype=BF16)
    out, lse = A.paged_attention(q, kp, vp, table, lengths)
    check_paged(A, q, (k[:200], k[200:]), (v[:200], v[200:]), out, lse, 0, 0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new", [None, [1, 0, 40, 7, 300], [0, 0, 0, 0, 0]])
@pytest.mark.parametrize("d", [1, 24, 128])
def test_append(A, dtype, new, d):
    lens, page, hk = [5, 0, 40, 100, 333], 16, 2
    kp, vp, table, lengths, _, _ = make_cache(lens, page, hk, d, dtype)
    kp, vp = torch.zeros_like(kp), torch.zeros_like(vp)
    counts = [1 if n else 0 for n in lens] if new is None else new
    rows = len(lens) if new is None else sum(new) + 3
    k, v = rnd(1, rows, hk + 1, d, dtype=dtype)[:, 1:], rnd(2, rows, hk, d, dtype=dtype)
    cu = None if new is None else torch.tensor([0] + list(itertools.accumulate(new)), dtype=torch.int32).cuda()
    wk, wv = kp.clone(), vp.clone()
    at = 0
    for i, (n, c) in enumerate(zip(lens, counts)):
        for j in range(c):
            pos = n - c + j
            src = i if new is None else at + j
            wk[table[i, pos // page], pos % page], wv[table[i, pos // page], pos % page] = k[src], v[src]
        at += c
    A.cache_append(k, v, kp, vp, table, lengths, cu)
    assert torch.equal(kp, wk) and torch.equal(vp, wv)


def test_append_drops_what_has_no_place(A):
    kp, vp, table, lengths, _, _ = make_cache([20, 20, 20, 20], 16, 1, 8, F32)
    kp, vp = torch.zeros_like(kp), torch.zeros_like(vp)
    k = rnd(1, 4, 1, 8)
    table[0, 1], table[1, 1] = -3, kp.shape[0]
    lengths[2], lengths[3] = 33, -5
    A.cache_append(k, k, kp, vp, table, lengths)
    assert (kp == 0).all() and (vp == 0).all()
    lengths[:] = torch.tensor([2, 1, 0, 0], dtype=torch.int32)               # fewer positions than rows: the last ones
    cu = torch.tensor([0, 3, 4, 4, 4], dtype=torch.int32).cuda()
    A.cache_append(k, k, kp, vp, table, lengths, cu)
    assert torch.equal(kp[table[0, 0], :2], k[1:3]) and torch.equal(vp[table[1, 0], :1], k[3:]) and int((kp != 0).sum()) == 24


# ------------------------------------------------------------------------------------------------ streams and graphs
def test_other_stream(A):
    q, k, v, do = (rnd(i, 1, 700, 4, 64, dtype=BF16) for i in (1, 2, 3, 4))
    out, lse = A.window_attention(q, k, v, 100, 4)
    grads = A.window_attention_backward(do, q, k, v, out, lse, 100, 4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    o2, l2 = A.window_attention(q, k, v, 100, 4, stream=s.cuda_stream)
    g2 = A.window_attention_backward(do, q, k, v, o2, l2, 100, 4, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(out, o2) and torch.equal(lse, l2) and all(torch.equal(a, b) for a, b in zip(grads, g2))
    with torch.cuda.stream(s):
        o3, _ = A.window_attention(q, k, v, 100, 4)
    s.synchronize()
    assert torch.equal(out, o3)


def test_graphs(A):
    """Forward, gradients, append and token attention captured together, replayed on new inputs with eager work between."""
    q, k, v, do = (rnd(i, 1, 300, 4, 64, dtype=BF16) for i in (1, 2, 3, 4))
    kp, vp, table, lengths, _, _ = make_cache([600, 40], 16, 2, 64, BF16)
    nk, nv, tq = rnd(5, 2, 2, 64, dtype=BF16), rnd(6, 2, 2, 64, dtype=BF16), rnd(7, 2, 8, 64, dtype=BF16)

    def step():
        out, lse = A.window_attention(q, k, v, 70, 4)
        grads = A.window_attention_backward(do, q, k, v, out, lse, 70, 4)
        A.cache_append(nk, nv, kp, vp, table, lengths)
        return (out, lse) + grads + A.paged_attention(tq, kp, vp, table, lengths)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                     # two graphs in one process, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    for i in range(4):
        for t in (q, k, v, do, nk, nv, tq):
            t.copy_(rnd(100 * i + t.numel() % 97, *t.shape, dtype=BF16))
        lengths.copy_(torch.tensor([600 - 7 * i, 40 - i], dtype=torch.int32))
        want = [x.clone() for x in step()]
        for g, res in graphs:
            for x in res:
                x.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, want))


# ------------------------------------------------------------------------------------------------ shapes of the blocks
LARGE = [
    # enough queries and keys for the large blocks, and the first keys' gradients split over chunks of queries
    (2200, 2200, 16, 8, 64, 200, 4, BF16), (1300, 1700, 32, 16, 128, 130, 40, F16), (1500, 1500, 16, 16, 40, 64, 100, BF16),
    (1200, 1200, 16, 16, 64, 100, 1, F32), (1100, 1100, 32, 32, 96, 0, 0, F16), (1030, 1030, 20, 20, 128, 70, 3, F32),
    # few keys, first keys split
    (2000, 2100, 4, 1, 64, 50, 33, BF16), (1000, 1000, 2, 2, 128, 100, 128, F32), (900, 900, 2, 1, 96, 60, 2, F16),
]


@pytest.mark.parametrize("case", LARGE, ids=str)
def test_block_shapes(A, case):
    nq, nk, h, hk, d, window, sinks, dtype = case
    q, k, v = rnd(1, nq, h, d, dtype=dtype), rnd(2, nk, hk, d, dtype=dtype), rnd(3, nk, hk, d, dtype=dtype)
    do = rnd(4, nq, h, d, dtype=dtype)
    out, lse = A.window_attention(q[None], k[None], v[None], window, sinks)
    got = A.window_attention_backward(do[None], q[None], k[None], v[None], out, lse, window, sinks)
    for kv in range(0, hk, max(1, hk // 3)):                     # a few key heads and their groups in float64
        group = slice(kv * (h // hk), (kv + 1) * (h // hk))
        r = O.attention(q[:, group], k[:, kv:kv + 1], v[:, kv:kv + 1], window, sinks)
        O.check("out", out[0][:, group], r["out"], r["tol_out"])
        O.check("lse", lse[0][:, group], r["lse"], r["tol_lse"])
        g = O.gradients(r, do[:, group])
        O.check("dq", got[0][0][:, group], g["dq"], g["tol_dq"])
        O.check("dk", got[1][0][:, kv:kv + 1], g["dk"], g["tol_dk"])
        O.check("dv", got[2][0][:, kv:kv + 1], g["dv"], g["tol_dv"])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_large_packed(A, dtype):
    """The split of the first keys in a ragged batch, with sequences shorter and longer than a chunk and rows behind."""
    lens, h, hk, d, window, sinks = [1500, 0, 3, 640, 900], 8, 4, 64, 100, 20
    n = sum(lens)
    q, do = rnd(1, n + 90, h, d, dtype=dtype), rnd(4, n + 90, h, d, dtype=dtype)
    k, v = rnd(2, n + 90, hk, d, dtype=dtype), rnd(3, n + 90, hk, d, dtype=dtype)
    cu = torch.tensor([0] + list(itertools.accumulate(lens)), dtype=torch.int32).cuda()
    out, lse = A.window_attention(q, k, v, window, sinks, cu_q=cu)
    got = A.window_attention_backward(do, q, k, v, out, lse, window, sinks, cu_q=cu)
    at = 0
    for m in lens:
        s = slice(at, at + m)
        r = O.attention(q[s], k[s], v[s], window, sinks)
        O.check("out", out[s], r["out"], r["tol_out"])
        g = O.gradients(r, do[s])
        for name, x in zip(("dq", "dk", "dv"), got):
            O.check(name, x[s], g[name], g["tol_" + name])
        at += m
    assert all((x[at:] == 0).all() for x in (out,) + got)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_masked_places_do_not_leak_in_large_blocks(A, dtype, value):
    n, h, hk, d, window, sinks, where = 1100, 32, 32, 64, 70, 2, 333
    base = [rnd(i, 1, n, h if i in (1, 4) else hk, d, dtype=dtype) for i in (1, 2, 3, 4)]
    seen = O.visible(n, n, window, sinks)
    rows, keys = ~seen[:, where], ~seen[where]
    run = lambda q, k, v, do: (lambda o, l: (o, l) + A.window_attention_backward(do, q, k, v, o, l, window, sinks))(
        *A.window_attention(q, k, v, window, sinks))
    ref = run(*base)
    for i in range(4):
        x = [t.clone() for t in base]
        x[i][0, where, :, 3] = value
        got = run(*x)
        if i in (1, 2):
            assert all(torch.equal(got[j][0][rows], ref[j][0][rows]) for j in (0, 1, 2))
        else:
            other = torch.arange(n) != where
            assert all(torch.equal(got[j][0][other], ref[j][0][other]) for j in (0, 2))
            assert all(torch.equal(got[j][0][keys], ref[j][0][keys]) for j in (3, 4))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_hidden_values_of_several_tiles(A, dtype):
    """Values that are not finite in tile after tile, some at the start and some at the end of what a block takes: every
    wave of a block has to take the careful way at the same place, each time."""
    n, h, hk, d, window, sinks = 420, 4, 2, 64, 48, 3
    base = [rnd(i, 1, n, h if i in (1, 4) else hk, d, dtype=dtype) for i in (1, 2, 3, 4)]
    at = torch.tensor([20, 64, 95, 127, 128, 161, 192, 255, 256, 300, 319])
    run = lambda q, k, v, do: (lambda o, l: (o, l) + A.window_attention_backward(do, q, k, v, o, l, window, sinks))(
        *A.window_attention(q, k, v, window, sinks))
    ref = run(*base)
    seen = O.visible(n, n, window, sinks)
    rows = ~seen[:, at].any(1)
    x = [t.clone() for t in base]
    x[1][:, at, :, 3] = x[2][:, at, :, 60] = math.nan
    first = run(*x)
    assert int(rows.sum()) > 60
    assert all(torch.equal(first[j][0][rows], ref[j][0][rows]) for j in (0, 1, 2))
    assert all(not torch.isfinite(first[j][0][~rows]).all(-1).any() for j in (0, 2))
    for _ in range(5):
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(run(*x), first))


@pytest.mark.parametrize("cuts", [(0, 900), (0, 1, 2, 900), (0, 880, 890, 900)], ids=str)
def test_first_keys_of_long_and_short_sequences(A, cuts):
    """The first keys' gradients where the mean length is on either side of what has their queries split."""
    n, h, hk, d, window, sinks = cuts[-1], 4, 2, 64, 40, 4
    q, k, v, do = (rnd(i, n, h if i in (1, 4) else hk, d, dtype=F16) for i in (1, 2, 3, 4))
    cu = torch.tensor(cuts, dtype=torch.int32).cuda()
    out, lse = A.window_attention(q, k, v, window, sinks, cu_q=cu)
    got = A.window_attention_backward(do, q, k, v, out, lse, window, sinks, cu_q=cu)
    for a, b in zip(cuts, cuts[1:]):
        s = slice(a, b)
        r = O.attention(q[s], k[s], v[s], window, sinks)
        O.check("out", out[s], r["out"], r["tol_out"])
        g = O.gradients(r, do[s])
        for name, x in zip(("dq", "dk", "dv"), got):
            O.check(name, x[s], g[name], g["tol_" + name])


def test_append_to_a_table_of_one_column(A):
    kp, vp = (torch.zeros(3, 4, 2, 8, device="cuda") for _ in range(2))
    k = rnd(1, 3, 2, 8)
    table = torch.tensor([[2], [0], [1]], dtype=torch.int32).cuda()
    A.cache_append(k, k, kp, vp, table, torch.tensor([4, 5, 0], dtype=torch.int32).cuda())      # the last, one too far, none
    assert torch.equal(kp[2, 3], k[0]) and torch.equal(vp[2, 3], k[0]) and int((kp != 0).sum()) == 16 == int((vp != 0).sum())


def test_integers_of_other_libraries(A):
    import numpy as np
    q = rnd(1, 1, 40, 2, 16)
    a, b = A.window_attention(q, q, q, 8, 2), A.window_attention(q, q, q, np.int64(8), np.int32(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# long and short sequences together: more than 64, more parts than one sequence may have, more sequences than parts are wanted
CUT = [
    ([9000] + [1 + 7 * i for i in range(69)], 4, 2, 64, 16, 0, 0), ([20000], 2, 1, 32, 64, 0, 0),
    ([300 - 3 * i for i in range(40)], 64, 64, 8, 16, 0, 0), ([6001, 0, 1, 2500, 63, 64, 65, 900], 24, 1, 128, 32, 0, 0),
    ([6001, 3, 4000, 1500] * 5, 8, 8, 80, 16, 1000, 40),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("case", CUT, ids=lambda c: str(c)[:40])
def test_paged_mixed_lengths(A, case, dtype):
    lens, h, hk, d, page, window, sinks = case
    kp, vp, table, lengths, ks, vs = make_cache(lens, page, hk, d, dtype)
    q = rnd(5, len(lens), h, d, dtype=dtype)
    out, lse = A.paged_attention(q, kp, vp, table, lengths, window, sinks)
    check_paged(A, q, ks, vs, out, lse, window, sinks)
    again, lse2 = A.paged_attention(q, kp, vp, table, lengths, window, sinks)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_paged_bad_length_among_long_ones(A):
    lens = [4000, 700, 2000]
    kp, vp, table, lengths, ks, vs = make_cache(lens, 16, 2, 64, BF16)
    q = rnd(5, 3, 4, 64, dtype=BF16)
    lengths[1] = -4
    out, lse = A.paged_attention(q, kp, vp, table, lengths)
    assert out[1].isnan().all() and lse[1].isnan().all()
    check_paged(A, q[::2], ks[::2], vs[::2], out[::2], lse[::2], 0, 0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_paged_infinite_value_in_the_last_part(A, dtype):
    lens = [1100]
    kp, vp, table, lengths, ks, vs = make_cache(lens, 16, 1, 64, dtype)
    q = rnd(5, 1, 2, 64, dtype=dtype)
    vp[table[0, 1099 // 16], 1099 % 16, 0, 5] = math.inf
    out, lse = A.paged_attention(q, kp, vp, table, lengths)
    assert (out[0, :, 5] == math.inf).all() and torch.isfinite(out[0, :, :5]).all() and torch.isfinite(lse).all()


def test_paged_graph_follows_the_lengths(A):
    """A captured call replayed as the sequences grow and shrink: the cut into parts is taken anew each time."""
    full = [5000, 300, 4000, 2500]
    kp, vp, table, lengths, ks, vs = make_cache(full, 32, 2, 64, BF16)
    q = rnd(5, 4, 8, 64, dtype=BF16)
    lengths[:] = 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        A.paged_attention(q, kp, vp, table, lengths)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = A.paged_attention(q, kp, vp, table, lengths)
    for now in ([1, 1, 1, 1], full, [0, 300, 17, 2500], [4999, 1, 0, 0], full):
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        check_paged(A, q, [k[:n] for k, n in zip(ks, now)], [v[:n] for v, n in zip(vs, now)], out, lse, 0, 0)
        eager, l2 = A.paged_attention(q, kp, vp, table, lengths)
        assert torch.equal(out, eager) and torch.equal(lse, l2)


def test_paged_on_two_streams(A):
    lens = [3000, 40, 900]
    kp, vp, table, lengths, ks, vs = make_cache(lens, 16, 2, 64, F16)
    qs = [rnd(i, 3, 4, 64, dtype=F16) for i in range(4)]
    want = [A.paged_attention(q, kp, vp, table, lengths) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = [A.paged_attention(q, kp, vp, table, lengths, stream=streams[i % 2].cuda_stream) for i, q in enumerate(qs)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
