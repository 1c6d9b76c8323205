"""The attention and 4-bit product libraries without a GPU: exports, what they refuse (before any device work), and the
float64 forms their GPU tests compare with."""
import ctypes as C
import re
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import attention_oracle as O

ROOT = Path(__file__).resolve().parents[1]
LIB = ROOT / "spmm-research_amd" / "lib"
P = 1 << 20                                              # an address that is aligned and never read


@pytest.mark.parametrize("header,lib,prefix,count", [("spmm_attn.h", "libspmm_attn.so", "attn", 7), ("spmm_q4.h", "libspmm_q4.so", "q4", 4)])
def test_exports(header, lib, prefix, count):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / header).read_text(), flags=re.S)
    names = sorted(set(re.findall(rf"\b(spmm_{prefix}_[a-z0-9_]+)\s*\(", text)))
    assert len(names) == count
    out = subprocess.run(["nm", "-D", "--defined-only", str(LIB / lib)], capture_output=True, text=True).stdout
    for n in names:
        assert re.search(rf"\bT {n}$", out, re.M), n
    r = subprocess.run([sys.executable, str(ROOT / "tools" / "check_fatbin.py"), str(LIB / lib)], capture_output=True, text=True)
    assert r.returncode == 0 and "missing 0" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("header", ["spmm_attn.h", "spmm_q4.h"])
def test_headers_are_c(header, tmp_path):
    src = tmp_path / "t.c"
    src.write_text(f'#include "{header}"\nint main(void) {{ return 0; }}\n')
    r = subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", f"-I{ROOT / 'include'}", "-c", str(src), "-o", str(tmp_path / "t.o")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


# ------------------------------------------------------------------------------------------------ attention, C ABI
def desc(A, **kw):
    base = dict(device=0, dtype=A.BF16, heads=4, kv_heads=2, dim=64, window=8, sinks=2, scale=0.1, batch=2, q_len=16, k_len=16,
                zero_rest=0, reserved=0)
    base.update(kw)
    return A._Desc(**base)


def rows(A, ptr=P, seq=16 * 256, row=256, head=64):
    return A._Rows(ptr, seq, row, head)


@pytest.fixture(scope="module")
def A():
    from spmm_amd import attention
    return attention


def window(A, d=None, cu=(None, None), lse=P, **kw):
    d = d if d is not None else desc(A)
    r = {n: kw.get(n, rows(A)) for n in ("q", "k", "v", "out")}
    return A.lib.spmm_attn_window(d, r["q"], r["k"], r["v"], cu[0], cu[1], r["out"], lse, None)


def grad(A, d=None, cu=(None, None), work=P, nbytes=1 << 20, **kw):
    d = d if d is not None else desc(A)
    r = {n: kw.get(n, rows(A)) for n in ("dout", "q", "k", "v", "out", "dq", "dk", "dv")}
    return A.lib.spmm_attn_window_grad(d, r["dout"], r["q"], r["k"], r["v"], r["out"], P, cu[0], cu[1], r["dq"], r["dk"], r["dv"],
                                       work, nbytes, None)


def pages(A, **kw):
    base = dict(k=P, v=P, pages=8, page_rows=16, k_page=16 * 128, k_row=128, k_head=64, v_page=16 * 128, v_row=128, v_head=64,
                table=P, table_cols=4, table_stride=4, lengths=P)
    base.update(kw)
    return A._Pages(**base)


def paged(A, d=None, p=None, longest=64, work=P, nbytes=1 << 20, **kw):
    return A.lib.spmm_attn_paged(d if d is not None else desc(A), kw.get("q", A._Rows(P, 256, 0, 64)),
                                 p if p is not None else pages(A), longest, kw.get("out", A._Rows(P, 256, 0, 64)), kw.get("lse", P),
                                 work, nbytes, None)


def append(A, d=None, p=None, cu=None, **kw):
    return A.lib.spmm_attn_append(d if d is not None else desc(A), kw.get("k", A._Rows(P, 0, 128, 64)), kw.get("v", A._Rows(P, 0, 128, 64)),
                                  cu, p if p is not None else pages(A), None)


needs_no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="valid arguments would run")


@needs_no_gpu
def test_valid_arguments_need_a_device(A):
    assert window(A) == grad(A) == paged(A) == append(A) == -4
    assert b"no HIP device" in A.lib.spmm_attn_last_error_detail()


BAD_DESC = [(dict(dtype=0), -1), (dict(dtype=4), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(heads=3), -1), (dict(heads=65536), -1),
            (dict(dim=0), -1), (dict(dim=129), -1), (dict(window=-1), -1), (dict(sinks=-1), -1), (dict(scale=float("nan")), -1),
            (dict(scale=float("inf")), -1), (dict(batch=-1), -1), (dict(q_len=-1), -1), (dict(k_len=-1), -1), (dict(zero_rest=2), -1),
            (dict(reserved=1), -1), (dict(batch=2 ** 31), -7), (dict(q_len=2 ** 31), -7), (dict(k_len=2 ** 40), -7)]


@pytest.mark.parametrize("bad,status", BAD_DESC, ids=str)
def test_bad_descriptions(A, bad, status):
    d = desc(A, **bad)
    n = C.c_size_t()
    assert window(A, d) == grad(A, d) == paged(A, d) == append(A, d) == status
    assert A.lib.spmm_attn_window_work(d, 0, n) == A.lib.spmm_attn_paged_work(d, 64, n) == status


def test_missing_description(A):
    n = C.c_size_t()
    assert A.lib.spmm_attn_window_work(None, 0, n) == -1 and A.lib.spmm_attn_window_work(desc(A), 0, None) == -1
    assert A.lib.spmm_attn_window(None, rows(A), rows(A), rows(A), None, None, rows(A), P, None) == -1


def test_bad_window_operands(A):
    for name in ("q", "k", "v", "out"):
        assert window(A, **{name: None}) == -1
        assert window(A, **{name: rows(A, ptr=None)}) == -1
        assert window(A, **{name: rows(A, ptr=P + 1)}) == -1                  # off its elements
        assert window(A, **{name: rows(A, row=-256)}) == -1
        assert window(A, **{name: rows(A, seq=2 ** 61)}) == -7
        assert name.encode() in A.lib.spmm_attn_last_error_detail()
    assert window(A, lse=None) == -1 and window(A, lse=P + 2) == -1
    assert window(A, cu=(P, None)) == -1 and window(A, cu=(None, P)) == -1 and window(A, cu=(P + 2, P)) == -1
    for bad in (dict(head=0), dict(head=63), dict(row=255), dict(seq=0), dict(seq=16 * 256 - 1)):     # rows that are written overlap
        assert window(A, out=rows(A, **bad)) == -1
        assert grad(A, dq=rows(A, **bad)) == -1
    # two key heads: a row spans 128, sixteen rows 256 * 15 + 128
    for bad in (dict(head=0), dict(head=63), dict(row=127), dict(seq=0), dict(seq=256 * 15 + 127)):
        assert grad(A, dk=rows(A, **bad)) == -1 and grad(A, dv=rows(A, **bad)) == -1
    for name in ("dout", "q", "k", "v", "out", "dq", "dk", "dv"):
        assert grad(A, **{name: None}) == -1 and grad(A, **{name: rows(A, ptr=None)}) == -1
    assert grad(A, work=None) == -1 and grad(A, work=P + 8) == -1 and grad(A, nbytes=2 * 16 * 4 * 8 - 1) == -1


def test_workspaces(A):
    n = C.c_size_t()
    assert A.lib.spmm_attn_window_work(desc(A, batch=3, q_len=7, heads=4), 0, n) == 0 and n.value == 3 * 7 * 4 * 8
    assert A.lib.spmm_attn_window_work(desc(A, batch=3, q_len=7, heads=4), 1, n) == 0 and n.value == 7 * 4 * 8
    assert A.lib.spmm_attn_window_work(desc(A, batch=2 ** 29, q_len=2 ** 29), 0, n) == -7
    assert A.lib.spmm_attn_paged_work(desc(A), -1, n) == -1 and A.lib.spmm_attn_paged_work(desc(A), 2 ** 31, n) == -1
    assert A.lib.spmm_attn_paged_work(desc(A, window=0), 10, n) == 0 and n.value == 0     # one part: nothing to join
    assert A.lib.spmm_attn_paged_work(desc(A, window=0), 100000, n) == 0 and n.value > 0


def test_empty_calls_do_nothing(A):
    assert window(A, desc(A, batch=0)) == 0 and window(A, desc(A, q_len=0), q=rows(A, ptr=None), out=rows(A, ptr=None), lse=None) == 0
    assert grad(A, desc(A, batch=0)) == 0 and paged(A, desc(A, batch=0)) == 0 and append(A, desc(A, batch=0)) == 0
    assert append(A, desc(A, q_len=0), cu=P, k=A._Rows(None, 0, 0, 0), v=A._Rows(None, 0, 0, 0)) == 0


def test_bad_pages(A):
    for bad, status in [(dict(pages=-1), -1), (dict(page_rows=0), -1), (dict(table_cols=-1), -1), (dict(table_stride=3), -1), (dict(table_stride=-4), -1),
                        (dict(pages=2 ** 33), -7), (dict(page_rows=2 ** 31), -7), (dict(k=None), -1), (dict(v=None), -1), (dict(table=None), -1),
                        (dict(lengths=None), -1), (dict(table=P + 1), -1), (dict(lengths=P + 2), -1), (dict(k=P + 1), -1), (dict(v_row=-128), -1),
                        (dict(k_page=2 ** 60), -7)]:
        assert paged(A, p=pages(A, **bad)) == append(A, p=pages(A, **bad)) == status, bad
    for bad in (dict(k_head=63), dict(v_row=127), dict(k_page=16 * 128 - 1), dict(v_page=0)):           # only what is written must not overlap
        assert append(A, p=pages(A, **bad)) == -1
    assert paged(A, q=None) == paged(A, out=None) == paged(A, lse=None) == paged(A, longest=-1) == -1
    assert paged(A, out=A._Rows(P, 0, 0, 64)) == -1 and paged(A, out=A._Rows(P, 256, 0, 10)) == -1
    d = desc(A, window=0)
    n = C.c_size_t()
    big = pages(A, table_cols=1000, table_stride=1000)
    assert A.lib.spmm_attn_paged_work(d, 16000, n) == 0
    assert paged(A, d, big, 16000, nbytes=n.value - 1) == paged(A, d, big, 16000, work=None) == paged(A, d, big, 16000, work=P + 4) == -1
    assert append(A, cu=P + 1) == append(A, k=None) == append(A, v=A._Rows(None, 0, 128, 64)) == -1


# ------------------------------------------------------------------------------------------------ Python
def test_python_refuses_host_tensors_and_wrong_types(A):
    t = torch.zeros(1, 4, 2, 8)
    with pytest.raises(ValueError, match="no CPU path"):
        A.window_attention(t, t, t)
    with pytest.raises(TypeError, match="torch tensor"):
        A.window_attention([1.0], t, t)
    with pytest.raises(ValueError, match="no CPU path"):
        A.paged_attention(t[0], t, t, t, t)
    with pytest.raises(ValueError, match="no CPU path"):
        A.cache_append(t[0], t[0], t, t, t, t)
    from spmm_amd import q4
    with pytest.raises(ValueError, match="no CPU path"):
        q4.Q4Format(torch.zeros(2, 2, dtype=torch.uint8), torch.zeros(2, 1))


# ------------------------------------------------------------------------------------------------ 4-bit, C ABI
def test_q4_refusals():
    from spmm_amd import q4
    L = q4.lib

    def d(**kw):
        base = dict(device=0, dtype=q4.F16, rows=100, cols=300, group=64, zeros=0)
        base.update(kw)
        return q4._Desc(**base)
    n = C.c_size_t()
    assert L.spmm_q4_layout_bytes(d(), n) == 0 and n.value == 7 * 3 * 1024 + 7 * 5 * 32 + 160          # scales end on 256 bytes
    assert L.spmm_q4_layout_bytes(d(zeros=1), n) == 0
    for bad, status in [(dict(dtype=0), -1), (dict(rows=-1), -1), (dict(cols=-1), -1), (dict(rows=2 ** 31), -7), (dict(cols=2 ** 31), -7), (dict(group=0), -1),
                        (dict(group=16), -1), (dict(group=96), -1), (dict(group=192), -1), (dict(group=-128), -1), (dict(zeros=2), -1)]:
        w = d(**bad)
        assert L.spmm_q4_layout_bytes(w, n) == status
        assert L.spmm_q4_layout(w, P, 150, P, 5, None, 0, P, 1 << 30, None) == status
        assert L.spmm_q4_matvec(w, P, P, 300, 1, P, 100, None) == status
    lay = lambda w=d(), packed=P, ps=150, s=P, ss=5, z=None, zs=0, dst=P, nb=1 << 30: L.spmm_q4_layout(w, packed, ps, s, ss, z, zs, dst, nb, None)
    assert lay(packed=None) == lay(s=None) == lay(s=P + 1) == lay(dst=None) == lay(dst=P + 16) == lay(nb=100) == lay(ps=-1) == lay(ss=-1) == -1
    assert lay(w=d(zeros=1)) == -1 and lay(z=P) == -1
    mv = lambda w=d(), lay=P, x=P, xs=300, t=1, y=P, ys=100: L.spmm_q4_matvec(w, lay, x, xs, t, y, ys, None)
    assert mv(lay=None) == mv(lay=P + 128) == mv(x=None) == mv(x=P + 1) == mv(y=None) == mv(y=P + 1) == mv(t=-1) == mv(xs=-1) == mv(t=2, ys=99) == -1
    assert mv(t=65536) == -7 and mv(t=0) == 0 and mv(w=d(rows=0)) == 0
    if not torch.cuda.is_available():
        assert mv() == lay() == -4


# ------------------------------------------------------------------------------------------------ the float64 forms themselves
def test_oracle_attention_against_loops():
    """The dense float64 form against a loop over the definition, its gradients against automatic differentiation."""
    g = torch.Generator().manual_seed(0)
    nq, nk, h, hk, d, window, sinks = 9, 13, 4, 2, 5, 4, 2
    q, k, v, do = (torch.randn(n, m, d, generator=g).double().requires_grad_() for n, m in ((nq, h), (nk, hk), (nk, hk), (nq, h)))
    outs = []
    for i in range(nq):
        p = i + nk - nq
        js = [j for j in range(nk) if j <= p and (p - j < window or j < sinks)]
        for a in range(h):
            w = torch.softmax(torch.stack([q[i, a] @ k[j, a // 2] * d ** -0.5 for j in js]), 0)
            outs.append(sum(w[n] * v[j, a // 2] for n, j in enumerate(js)))
    out = torch.stack(outs).reshape(nq, h, d)
    r = O.attention(q, k, v, window, sinks)
    assert (r["out"] - out).abs().max() < 1e-13
    got = O.gradients(r, do)
    for name, want in zip(("dq", "dk", "dv"), torch.autograd.grad((out * do).sum(), (q, k, v))):
        assert (got[name] - want).abs().max() < 1e-12


def test_oracle_notices_a_wrong_result():
    """The bounds are tight enough to see one key too many or too few."""
    g = torch.Generator().manual_seed(0)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        q, k, v = (torch.randn(40, 2, 64, generator=g).to(dtype) for _ in range(3))
        r = O.attention(q, k, v, 10, 2)
        for other in (O.attention(q, k, v, 11, 2), O.attention(q, k, v, 10, 1)):
            with pytest.raises(AssertionError):
                O.check("out", other["out"].to(dtype), r["out"], r["tol_out"])
        O.check("out", r["out"].to(dtype), r["out"], r["tol_out"])
