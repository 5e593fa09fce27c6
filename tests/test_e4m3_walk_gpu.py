"""Rows in 8 bits of prompts: many long rows, which blocks that stay walk out of a ring of bulk copies, and the sizes next to where that form ends."""
import pytest
import torch

from tests.test_e4m3_gpu import HALF, check_rows, norm64, norm_rel, rand

pytestmark = pytest.mark.gpu


def silu_of(x, block=0):
    """silu(gate) * up in float64."""
    inter = x.shape[1] // 2
    at = torch.arange(inter, device=x.device)
    gate_at = at // block * 2 * block + at % block if block else at
    gate, up = x.double()[:, gate_at], x.double()[:, gate_at + (block or inter)]
    return gate * torch.sigmoid(gate) * up


# two rows of inputs take 220 KB of shared memory at 28,160 numbers of 16 bits (gate and up) and 14,080 of 32: the longest rows that are walked
@pytest.mark.parametrize("dtype,edge", [(torch.bfloat16, 28160), (torch.float32, 14080)])
@pytest.mark.parametrize("beyond", [0, 8, 128, 248, 256, 264])
def test_gates_next_to_the_longest_row_that_is_walked(kernels, dtype, edge, beyond):
    inter = edge + beyond if dtype == torch.bfloat16 else edge + beyond // 16 * 8
    x = rand((300, 2 * inter), dtype, 3, 3.0)
    q, scale = kernels.silu_mul_e4m3(x)
    check_rows(q, scale, silu_of(x), 9 * HALF, f"silu_mul of {inter}")
    few, few_scale = kernels.silu_mul_e4m3(x[200:].contiguous())          # a block a row
    assert torch.equal(q[200:].view(torch.uint8), few.view(torch.uint8)) and torch.equal(scale[200:], few_scale)


@pytest.mark.parametrize("hidden", [14080, 14088, 14200, 14208, 14216])
def test_norms_next_to_the_longest_row_that_is_walked(kernels, hidden):
    x, res, w = rand((300, hidden), torch.float32, 1, 3.0), rand((300, hidden), torch.float32, 2), 1 + rand((hidden,), torch.float32, 3, 0.1)
    s = x + res
    q, scale = kernels.add_rms_norm_e4m3(x, res, w, 1e-5)
    assert torch.equal(res, s)
    check_rows(q, scale, norm64(s, w, 1e-5), norm_rel(hidden), f"add_norm of {hidden}")


def turns(rows, per_processor):
    """Rows that give every block that stays (``per_processor`` of them) more than four turns, and some blocks one more than others."""
    at_once = torch.cuda.get_device_properties(0).multi_processor_count * per_processor
    assert rows > 4 * at_once and rows % at_once, f"{rows} rows, {at_once} blocks"


# hidden sizes whose blocks have one, part of one and two vectors of eight a thread; every block's ring of two rows goes round more than twice
@pytest.mark.parametrize("dtype,stream", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,hidden,per_processor", [(5003, 4096, 4), (2100, 8192, 2), (700, 12288, 1), (650, 9000, 1), (300, 16384, 0)])
def test_norms_of_prompts(kernels, dtype, stream, rows, hidden, per_processor):
    turns(rows, per_processor) if per_processor else None
    eps = 1e-5
    x, res = rand((rows, hidden), dtype, 2, 3.0), rand((rows, hidden), stream, 3, 2.0)
    w = 1 + rand((hidden,), torch.bfloat16, 4, 0.1)
    rel, half = norm_rel(hidden), torch.finfo(dtype).eps / 2
    s = (x.float() + res.float()).to(stream)
    v = norm64(s, w, eps)
    run = res.clone()
    q, scale, kept = kernels.add_rms_norm_e4m3(x, run, w, eps, keep=True)
    assert torch.equal(run, s), "the stream is the sum, rounded once"
    check_rows(q, scale, v, rel, "add_norm")
    assert kept.dtype == dtype and bool(((kept.double() - v).abs() <= (rel + half) * v.abs()).all())
    run = res.clone()
    again = kernels.add_rms_norm_e4m3(x, run, w, eps)
    assert torch.equal(run, s) and torch.equal(again[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(again[1], scale)


@pytest.mark.parametrize("dtype,stream", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("rows,hidden,picked", [(3000, 4096, 4500), (500, 12288, 700)])
def test_norms_of_gathered_rows_of_prompts(kernels, dtype, stream, rows, hidden, picked):
    """Any order, the same row again and again, the first and the last; the stream stays as it is."""
    eps = 1e-5
    x, res = rand((rows, hidden), dtype, 2, 3.0), rand((rows, hidden), stream, 3, 2.0)
    w = 1 + rand((hidden,), torch.float32, 4, 0.1)
    sel = torch.randint(0, rows, (picked,), dtype=torch.int32, generator=torch.Generator().manual_seed(5))
    sel[0], sel[1], sel[7:20] = rows - 1, 0, 11
    run = res.clone()
    q, scale, kept = kernels.add_rms_norm_e4m3(x, run, w, eps, sel.cuda(), keep=True)
    assert torch.equal(run, res)
    v = norm64((x.float() + res.float()).to(stream), w, eps)[sel.long().cuda()]
    check_rows(q, scale, v, norm_rel(hidden), "add_norm rows")
    assert bool(((kept.double() - v).abs() <= (norm_rel(hidden) + torch.finfo(dtype).eps / 2) * v.abs()).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,inter,block,per_processor", [(4203, 4096, 0, 0), (4203, 4096, 128, 0), (1201, 12288, 0, 2), (1201, 12288, 128, 2), (1201, 12288, 24, 2),
                                                              (2049, 8192, 2048, 0), (301, 25600, 0, 0), (301, 25600, 25600, 0), (650, 8200, 0, 0)])
def test_gates_of_prompts(kernels, dtype, tokens, inter, block, per_processor):
    """Gate and up one behind the other and in blocks, of powers of two and others."""
    turns(tokens, per_processor) if per_processor else None
    x = rand((tokens, 2 * inter), dtype, 5, 3.0)
    x[0, 0], x[0, -1] = -200.0, 100.0
    q, scale = kernels.silu_mul_e4m3(x, block)
    check_rows(q, scale, silu_of(x, block), 9 * HALF, "silu_mul")
    few, few_scale = kernels.silu_mul_e4m3(x[-200:].contiguous(), block)          # a block a row
    assert torch.equal(q[-200:].view(torch.uint8), few.view(torch.uint8)) and torch.equal(scale[-200:], few_scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [8200, 12344, 16384, 16392, 25600, 32768, 32776])
def test_long_rows_a_block_each(kernels, dtype, cols):
    """Rows of two and of four vectors of eight a thread, and the first beyond them, for few rows and for the most that are not walked."""
    for rows in (3, 295):
        x, res = rand((rows, cols), dtype, 1, 3.0), rand((rows, cols), dtype, 2)
        check_rows(*kernels.quantise_e4m3(x), x.double(), 0.0, "quantise")
        w = 1 + rand((cols,), torch.bfloat16, 3, 0.1)
        check_rows(*kernels.rms_norm_e4m3(x, w, 1e-5), norm64(x, w, 1e-5), norm_rel(cols), "norm")
        s = (x.float() + res.float()).to(dtype)
        check_rows(*kernels.add_rms_norm_e4m3(x, res, w, 1e-5), norm64(s, w, 1e-5), norm_rel(cols), "add_norm")
        assert torch.equal(res, s)
        wide = x.float().clone()
        check_rows(*kernels.add_rms_norm_e4m3(x, wide, w, 1e-5), norm64(x.float() + x.float(), w, 1e-5), norm_rel(cols), "add_norm over 32 bits")
    check_rows(*kernels.quantise_e4m3(rand((1200, cols), dtype, 7)), rand((1200, cols), dtype, 7).double(), 0.0, "quantise of many rows")


def test_a_walked_rows_nan_stays_in_its_row(kernels):
    """A row that holds a NaN or an infinity in the middle of the walk; its block's later rows, its ring's slot among them, are as without it."""
    for cols, call in ((12288, lambda v: kernels.silu_mul_e4m3(v.repeat(1, 2))),
                       (12288, lambda v: kernels.add_rms_norm_e4m3(v, torch.ones_like(v), torch.ones(12288, device="cuda"), 1e-6))):
        x = rand((900, cols), torch.bfloat16, 1)
        clean, clean_scale = call(x)
        x[148, 5], x[451, 9000] = float("nan"), float("inf")
        q, scale = call(x)
        assert not torch.isfinite(scale[[148, 451]] * q[[148, 451]].float().abs().amax(1)).any()
        keep = [i for i in range(900) if i not in (148, 451)]
        assert torch.equal(q[keep].view(torch.uint8), clean[keep].view(torch.uint8)) and torch.equal(scale[keep], clean_scale[keep])


def test_walks_on_two_streams_and_in_graphs(kernels):
    """Two walks at once, and two captured ones that are replayed in turn on new inputs."""
    w = torch.ones(4096, dtype=torch.bfloat16, device="cuda")
    xs = [rand((4500, 4096), torch.bfloat16, i, 2.0) for i in range(4)]
    wants = [(kernels.add_rms_norm_e4m3(x, torch.zeros_like(x), w, 1e-6), kernels.silu_mul_e4m3(x.repeat(1, 2))) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], {}
    for i, x in enumerate(xs):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = kernels.add_rms_norm_e4m3(x, torch.zeros_like(x), w, 1e-6), kernels.silu_mul_e4m3(x.repeat(1, 2))
    torch.cuda.synchronize()
    statics, graphs = [x.clone() for x in xs[:2]], []
    for x in statics:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = kernels.add_rms_norm_e4m3(x, torch.zeros_like(x), w, 1e-6), kernels.silu_mul_e4m3(x.repeat(1, 2))
        graphs.append((g, out))

    def same(a, b):
        return all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip((*a[0], *a[1]), (*b[0], *b[1])))

    assert all(same(got[i], wants[i]) for i in range(4))
    for turn in (0, 2):
        for i in range(2):
            statics[i].copy_(xs[turn + i])
        for i in (0, 1, 0):
            graphs[i][0].replay()
        torch.cuda.synchronize()
        assert all(same(graphs[i][1], wants[turn + i]) for i in range(2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,inter", [(5, 44), (5, 96), (2, 9000), (300, 12288)])
def test_gates_far_below_zero_beside_large_values(kernels, dtype, tokens, inter):
    """exp(-g) is up to 2^128 there, and its reciprocal less than the least normal number; the product with up is an ordinary number. Every form of the kernel."""
    g = torch.linspace(-88.5, -84.0, inter, device="cuda").to(dtype)
    u = torch.full((inter,), 3e38, device="cuda").to(dtype)
    x = torch.cat([g, u]).repeat(tokens, 1).contiguous()
    want = silu_of(x)
    assert float(want.abs().min()) > 90
    q, scale, kept = kernels.silu_mul_e4m3(x, keep=True)
    check_rows(q, scale, want, 9 * HALF, "silu_mul")
    assert bool(((kept.double() - want).abs() <= (9 * HALF + torch.finfo(dtype).eps / 2) * want.abs()).all())
