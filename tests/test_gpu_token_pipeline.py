"""The token pipeline on the GPU: 4-bit projections, cache and attention together, against float64."""
import pytest
import torch

import attention_oracle as O

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HEADS, KV, D, WIDTH, PAGE, WINDOW, SINKS = 8, 2, 64, 192, 16, 40, 3


@pytest.fixture(scope="module")
def mods():
    assert torch.cuda.is_available(), "gpu tests need a HIP device"
    from spmm_amd import pipeline, q4
    return pipeline, q4


def weights(q4, rows, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    packed = torch.randint(0, 256, (rows, WIDTH // 2), generator=g, dtype=torch.uint8).cuda()
    scales = (torch.rand(rows, WIDTH // 64, generator=g) * 0.02 + 0.005).to(dtype).cuda()
    return q4.Q4Format(packed, scales, group=64)


def make(mods, dtype, pages=40):
    pipeline, q4 = mods
    w = [weights(q4, n * D, dtype, i) for i, n in enumerate((HEADS, KV, KV))]
    return pipeline.TokenPipeline(*w, HEADS, KV, pages, PAGE, WINDOW, SINKS)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_prompt_and_steps(mods, dtype):
    """Prompts of 70, 1 and 33 tokens, then ten tokens each: every token's output is the attention of the projections so
    far, of which the float64 form gets the same (rounded) rows."""
    p = make(mods, dtype)
    lens, new = [70, 1, 33], 10
    g = torch.Generator().manual_seed(5)
    table = torch.randperm(40, generator=g)[:3 * 6].reshape(3, 6).int().cuda()
    xs = [torch.randn(n + new, WIDTH, generator=g).to(dtype).cuda() for n in lens]
    cu = torch.tensor([0, 70, 71, 104], dtype=torch.int32).cuda()
    lengths = torch.tensor(lens, dtype=torch.int32).cuda()
    out = p.prompt(torch.cat([x[:n] for x, n in zip(xs, lens)]), cu, table, lengths)
    outs = [[o] for o in out.split(lens)]
    for i in range(new):
        lengths += 1
        o = p.step(torch.stack([x[n + i] for x, n in zip(xs, lens)]), table, lengths, max_length=96)
        for j in range(3):
            outs[j].append(o[j:j + 1])
    for x, o, n in zip(xs, outs, lens):
        q, k, v = (p.w[t].matvec(x).view(n + new, -1, D) for t in "QKV")
        r = O.attention(q, k, v, WINDOW, SINKS)
        O.check("out", torch.cat(o).view(n + new, HEADS, D), r["out"], r["tol_out"])


def test_step_in_a_graph(mods):
    """One captured step serves every token: the table, the lengths and x are its inputs."""
    p, e = make(mods, torch.bfloat16), make(mods, torch.bfloat16)
    table = torch.arange(24, dtype=torch.int32).reshape(4, 6).cuda()
    lengths = torch.zeros(4, dtype=torch.int32).cuda()
    x = torch.zeros(4, WIDTH, dtype=torch.bfloat16).cuda()
    p.step(x, table, lengths, max_length=96)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = p.step(x, table, lengths, max_length=96)
    p.k_pages.zero_(), p.v_pages.zero_()
    for i in range(50):
        x.copy_(torch.randn(4, WIDTH, generator=torch.Generator().manual_seed(i)))
        lengths.copy_(torch.tensor([i + 1, i + 1, 0, max(0, i - 20)], dtype=torch.int32))     # one padded, one that joins later
        graph.replay()
        want = e.step(x, table, lengths, max_length=96)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert (out[2] == 0).all()


def test_refusals(mods):
    pipeline, q4 = mods
    w = [weights(q4, n * D, torch.float16, i) for i, n in enumerate((HEADS, KV, KV))]
    other = weights(q4, KV * D, torch.bfloat16, 1)
    for args in ((w[0], w[1], other, HEADS, KV), (w[0], w[1], w[2], HEADS, 4), (w[0], w[1], w[2], 7, 1), (w[0], w[0], w[2], HEADS, KV),
                 (w[0], w[1], w[2], 0, 1)):
        with pytest.raises(ValueError):
            pipeline.TokenPipeline(*args, pages=4)
