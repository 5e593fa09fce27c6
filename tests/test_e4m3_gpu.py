"""Rows in 8 bits (the residual's addition with the norm, silu(gate) * up, rows as they are) and the product that takes them, against the
definitions in float64.

A row's scale comes from one division (half a unit in the 24th bit) of a largest magnitude that is as far off as the row's numbers are (``rel``). A
number in 8 bits is the one nearest to v / scale, unless v / scale lies within that error of the middle between two."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F64, E4M3 = torch.float64, torch.float8_e4m3fn
HALF = 2.0 ** -24                 # float32: half a step, relative to the value
TOP, LEAST = 448.0, 2.0 ** -126


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def nearest(v):
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def check_rows(q, scale, v, rel, what):
    """q and scale against rows v in float64 that are known to ``rel``."""
    assert q.dtype == E4M3 and scale.dtype == torch.float32 and q.shape == v.shape and scale.shape == v.shape[:-1]
    want = (v.abs().amax(-1) / TOP).clamp_min(LEAST)
    off = float(((scale.double() - want).abs() / want).max())
    assert off <= rel + 2 * HALF, f"{what}: a scale is {off:.2e} off"
    ratio = v / scale.double()[..., None]
    got, ref = q.double(), nearest(ratio)
    middle = (got + ref) / 2
    # the quotient is formed from a reciprocal with one correction: two half steps more
    wrong = (got != ref) & ((ratio - middle).abs() > (rel + 4 * HALF) * ratio.abs())
    assert not bool(wrong.any()), f"{what}: {int(wrong.sum())} of {got.numel()} numbers are not the nearest"
    assert float((got != ref).double().mean()) < 0.01 or got.numel() < 1000, f"{what}: more than one number in a hundred lies at a middle"


def norm64(s, w, eps):
    s = s.double()
    return s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * w.double()


def norm_rel(hidden):
    """How far a 32-bit norm may be: the mean square's sum (at most hidden / 32 additions in a row a thread, then the tree), under the square
    root; the root, the quotient and two products."""
    return HALF * ((hidden / 32 + 16) / 2 + 6)


ROWS = [(1, 1), (1, 7), (3, 44), (5, 1000), (2, 1111), (9, 4096), (3, 5120), (2, 8192), (1100, 256), (1300, 4096), (2, 40000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", ROWS)
def test_quantise(kernels, dtype, rows, cols):
    x = rand((rows, cols), dtype, rows + cols, 3.0)
    x[rows // 2] *= 100
    q, scale = kernels.quantise_e4m3(x)
    check_rows(q, scale, x.double(), 0.0, "quantise")
    wide = rand((rows, cols + 24), dtype, 5)
    wide[:, 8:8 + cols] = x
    q2, scale2 = kernels.quantise_e4m3(wide[:, 8:8 + cols])      # rows that lie apart
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(scale2, scale)


def test_quantise_every_tie(kernels):
    """Every number of e4m3, every middle between two of them and their neighbours, with a scale of one."""
    top = torch.arange(0, 127, dtype=torch.uint8).view(E4M3).double()
    mid = (top[1:] + top[:-1]) / 2
    v = torch.cat([top, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    v = torch.cat([v, -v, torch.tensor([TOP], dtype=F64)]).float().cuda()
    q, scale = kernels.quantise_e4m3(v[None])
    assert float(scale[0]) == 1.0
    assert torch.equal(q.double()[0], nearest(v.double()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_zeros_and_the_least_and_largest_numbers(kernels, dtype):
    x = rand((6, 96), dtype, 8)
    x[0] = 0
    x[1] *= 1e-38 if dtype == torch.bfloat16 else 1e-42
    x[2] *= 1e37
    x[4, 3], x[5, 7] = float("inf"), float("nan")
    q, scale = kernels.quantise_e4m3(x)
    assert float(scale[0]) == LEAST and not bool(q[0].double().any())
    check_rows(q[:4], scale[:4], x[:4].double(), 0.0, "extremes")
    assert not torch.isfinite(scale[4:]).any()
    w, w_scale = kernels.quantise_e4m3(rand((32, 96), torch.bfloat16, 9))
    y = kernels.gemm_e4m3(q, scale, w, w_scale, torch.float32)
    assert torch.isnan(y[4:]).all() and torch.isfinite(y[:4]).all()       # the other rows keep their values


@pytest.mark.parametrize("dtype,stream", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,hidden", ROWS)
def test_norms(kernels, dtype, stream, wdtype, rows, hidden):
    eps = 1e-5
    x, res = rand((rows, hidden), dtype, 2, 3.0), rand((rows, hidden), stream, 3, 2.0)
    w = (1 + 0.1 * torch.randn(hidden, generator=torch.Generator().manual_seed(4))).to(wdtype).cuda()
    rel, half = norm_rel(hidden), torch.finfo(dtype).eps / 2

    def kept_ok(kept, v):
        assert kept.dtype == dtype and bool(((kept.double() - v).abs() <= (rel + half) * v.abs()).all())

    v = norm64(x, w, eps)
    q, scale = kernels.rms_norm_e4m3(x, w, eps)
    check_rows(q, scale, v, rel, "norm")
    q2, scale2, kept = kernels.rms_norm_e4m3(x, w, eps, keep=True)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(scale, scale2)
    kept_ok(kept, v)

    s = (x.float() + res.float()).to(stream)     # rounded once, to the stream's type
    v = norm64(s, w, eps)
    run = res.clone()
    q, scale, kept = kernels.add_rms_norm_e4m3(x, run, w, eps, keep=True)
    assert torch.equal(run, s)
    check_rows(q, scale, v, rel, "add_norm")
    kept_ok(kept, v)
    sel = torch.tensor([rows - 1, 0, 0], dtype=torch.int32).cuda()
    run = res.clone()
    q, scale = kernels.add_rms_norm_e4m3(x, run, w, eps, sel)
    assert torch.equal(run, res), "with gathered rows the residual stays as it is"
    check_rows(q, scale, v[[rows - 1, 0, 0]], rel, "add_norm rows")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,inter,block", [(1, 1, 0), (3, 100, 0), (17, 1111, 0), (2, 256, 128), (5, 384, 8), (16, 12288, 0), (3, 12288, 128),
                                                (1500, 512, 128), (2, 25600, 128), (1, 40000, 0)])
def test_silu_mul(kernels, dtype, tokens, inter, block):
    x = rand((tokens, 2 * inter), dtype, 5, 3.0)
    x[0, 0], x[0, -1] = -200.0, 100.0            # exp(200) is beyond float32
    at = torch.arange(inter, device="cuda")
    gate_at = at // block * 2 * block + at % block if block else at
    gate, up = x.double()[:, gate_at], x.double()[:, gate_at + (block or inter)]
    q, scale = kernels.silu_mul_e4m3(x, block)
    # In half steps (2^-24): expf is within 2 units of its last place, 4, and counts by exp(-g) / (1 + exp(-g)) < 1; the sum rounds, 1; its approximate
    # reciprocal is within a unit, 2; two products round, 2: 9 together. A gate far below zero gives a denormal or zero where the formula gives less
    # than the least number, which the 8 bits do not see.
    check_rows(q, scale, gate * torch.sigmoid(gate) * up, 9 * HALF, "silu_mul")


SIZES = [(1, 1, 1), (1, 70, 50), (3, 64, 16), (5, 130, 32), (1, 4096, 4096), (8, 129, 208), (16, 1000, 1024), (17, 24, 4112), (31, 6144, 2048), (33, 257, 144),
         (64, 2048, 5120), (65, 128, 128), (100, 300, 176), (129, 513, 2064), (256, 1024, 1024), (333, 6144, 1024), (512, 4096, 512), (700, 1111, 1040),
         (1025, 520, 16), (2048, 2048, 2048), (4, 100, 333)]


def product_check(got, q, q_scale, w, w_scale, what):
    """32-bit sums of exact products: each of the k additions is off by at most a step (the tensor cores cut off) of a sum no larger than that of the
    magnitudes; the two scales and the output round once each."""
    rows, cols = q.double() * q_scale.double()[:, None], w.double() * w_scale.double()[:, None]
    want = rows @ cols.t()
    bound = (torch.finfo(got.dtype).eps / 2 + 3 * HALF) * want.abs() + q.shape[1] * 2 * HALF * (rows.abs() @ cols.abs().t())
    worst = float(((got.double() - want).abs() / bound.clamp_min(1e-300)).max())
    print(f"MEASURED {what}: {worst:.3f} of the bound")
    assert worst <= 1.0, f"{what}: {worst} times the bound"


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(kernels, out, m, n, k):
    q, q_scale = kernels.quantise_e4m3(rand((m, k), torch.float32, 6))
    w, w_scale = kernels.quantise_e4m3(rand((n, k), torch.float32, 7, 0.02))
    got = kernels.gemm_e4m3(q, q_scale, w, w_scale, out)
    assert got.shape == (m, n) and got.dtype == out
    product_check(got, q, q_scale, w, w_scale, f"product {m} x {n} x {k}")
    again = kernels.gemm_e4m3(q, q_scale, w, w_scale, out)
    assert torch.equal(got, again), "the same bits on every run"


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 17, 1024), (8, 300, 1040), (3, 2049, 1536), (8, 4100, 2032), (6, 15000, 1040), (7, 16300, 2048), (2, 12001, 4080), (8, 26100, 528),
                                   (9, 33, 1024), (16, 9000, 528), (16, 9500, 1008), (11, 520, 2048), (13, 4700, 4096), (9, 100, 3600), (16, 4800, 2064), (10, 40000, 272)])
def test_product_of_a_handful_of_rows(kernels, out, m, n, k):
    """Both numbers of rows, the three depths of k with ends inside a block, strips that all run at once, that take turns, and one more than there are."""
    q, q_scale = kernels.quantise_e4m3(rand((m, k), torch.float32, 8))
    w, w_scale = kernels.quantise_e4m3(rand((n, k), torch.float32, 9, 0.02))
    got = kernels.gemm_e4m3(q, q_scale, w, w_scale, out)
    product_check(got, q, q_scale, w, w_scale, f"product {m} x {n} x {k}")
    assert torch.equal(got, kernels.gemm_e4m3(q, q_scale, w, w_scale, out))


@pytest.mark.parametrize("m,n,k", [(2, 5000, 12288), (7, 300, 8208), (30, 4100, 9008), (64, 20000, 8320), (90, 264, 16384), (300, 2050, 8208), (520, 4096, 8448),
                                   (1000, 4096, 14336), (2500, 4100, 8208), (4000, 72, 10240)])
def test_product_of_a_long_k(kernels, m, n, k):
    """Tiles, pairs and strips that a processor meets more than once, with two sums a tile; the errors together are below 2^-20 of the outputs."""
    q, q_scale = kernels.quantise_e4m3(rand((m, k), torch.float32, 8))
    w, w_scale = kernels.quantise_e4m3(rand((n, k), torch.float32, 9, 0.02))
    got = kernels.gemm_e4m3(q, q_scale, w, w_scale, torch.float32)
    product_check(got, q, q_scale, w, w_scale, f"product {m} x {n} x {k}")
    want = (q.double() @ w.double().t()) * q_scale.double()[:, None] * w_scale.double()
    assert (got.double() - want).norm() <= 2.0 ** -20 * want.norm()
    assert torch.equal(got, kernels.gemm_e4m3(q, q_scale, w, w_scale, torch.float32))
    product_check(kernels.gemm_e4m3(q, q_scale, w, w_scale, torch.bfloat16), q, q_scale, w, w_scale, f"product {m} x {n} x {k}, bfloat16")


@pytest.mark.parametrize("m,n,k,pad", [(9, 200, 256, 16), (9, 200, 256, 3), (200, 384, 512, 48), (40, 256, 96, 1)])
def test_product_of_rows_that_lie_apart(kernels, m, n, k, pad):
    q, q_scale = kernels.quantise_e4m3(rand((m, k + pad), torch.float32, 6))
    w, w_scale = kernels.quantise_e4m3(rand((n, k + pad), torch.float32, 7))
    for at in (0, pad):
        qv, wv = q[:, at:at + k], w[:, at:at + k]
        product_check(kernels.gemm_e4m3(qv, q_scale, wv, w_scale, torch.float32), qv, q_scale, wv, w_scale, "rows apart")


def test_product_keeps_a_rows_nan_to_itself(kernels):
    for m in (5, 40, 300):
        q, q_scale = kernels.quantise_e4m3(rand((m, 512), torch.float32, 6))
        w, w_scale = kernels.quantise_e4m3(rand((384, 512), torch.float32, 7))
        clean = kernels.gemm_e4m3(q, q_scale, w, w_scale)
        bytes_ = q.view(torch.uint8)
        bytes_[2, 100] = 0x7F                      # NaN
        q_scale[3] = float("inf")
        got = kernels.gemm_e4m3(q, q_scale, w, w_scale)
        assert torch.isnan(got[2]).all() and not torch.isfinite(got[3]).any()
        keep = [i for i in range(m) if i not in (2, 3)]
        assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("m", [4, 48, 300])
def test_a_weight_is_multiplied_right_after_it_is_quantised(kernels, m):
    """A product reads its weight ahead of the wait for the kernel in front, which here is the one that writes it."""
    q, q_scale = kernels.quantise_e4m3(rand((m, 4096), torch.float32, 1))
    stored = [rand((4096, 4096), torch.bfloat16, 10 + i) for i in range(4)]
    wants = []
    for w in stored:
        made = kernels.quantise_e4m3(w)
        torch.cuda.synchronize()
        wants.append(kernels.gemm_e4m3(q, q_scale, *made))
        del made
    torch.cuda.synchronize()
    for _ in range(5):
        for w, want in zip(stored, wants):
            assert torch.equal(kernels.gemm_e4m3(q, q_scale, *kernels.quantise_e4m3(w)), want)


def test_more_rows_than_a_grid_has_in_its_second_direction(kernels):
    """70,000 rows of the row kernels and of the products' forms, the last rows as well as the first."""
    x = rand((70000, 64), torch.bfloat16, 1)
    q, scale = kernels.quantise_e4m3(x)
    check_rows(q, scale, x.double(), 0.0, "quantise")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    for name, got in (("norm", kernels.rms_norm_e4m3(x, w, 1e-6)), ("silu_mul", kernels.silu_mul_e4m3(x))):
        few = kernels.rms_norm_e4m3(x[-70:], w, 1e-6) if name == "norm" else kernels.silu_mul_e4m3(x[-70:])
        assert torch.equal(got[0][-70:].view(torch.uint8), few[0].view(torch.uint8)) and torch.equal(got[1][-70:], few[1]), name
    wq, ws = kernels.quantise_e4m3(rand((40, 64), torch.float32, 2))
    product_check(kernels.gemm_e4m3(q, scale, wq, ws), q, scale, wq, ws, "70,000 rows")
    odd, odd_scale = kernels.quantise_e4m3(x[:, :50].contiguous())
    wq, ws = kernels.quantise_e4m3(rand((4, 50), torch.float32, 2))
    product_check(kernels.gemm_e4m3(odd, odd_scale, wq, ws), odd, odd_scale, wq, ws, "70,000 rows of any size")
    product_check(kernels.gemm_e4m3(wq, ws, odd, odd_scale), wq, ws, odd, odd_scale, "70,000 columns of any size")


@pytest.mark.parametrize("m", [5, 12, 200])
@pytest.mark.parametrize("k", [32784, 32785])
def test_a_weight_beyond_32_bits(kernels, m, k):
    """Rows of a weight that lie more than 2 ** 31 numbers behind its first, and of the rows that it is made from."""
    n = 66000
    w = torch.randint(0, 0x40, (n, k), dtype=torch.uint8, device="cuda").view(E4M3)
    w_scale = torch.ones(n, device="cuda")
    q, q_scale = kernels.quantise_e4m3(rand((m, k), torch.float32, 1))
    product_check(kernels.gemm_e4m3(q, q_scale, w, w_scale)[:, -300:], q, q_scale, w[-300:], w_scale[-300:], f"product {m} x {n} x {k}")
    if m == 5:
        x = w.to(torch.bfloat16)
        got, scale = kernels.quantise_e4m3(x)
        few = kernels.quantise_e4m3(x[-9:].clone())
        assert torch.equal(got[-9:].view(torch.uint8), few[0].view(torch.uint8)) and torch.equal(scale[-9:], few[1])


def test_rows_of_more_than_two_dimensions(kernels):
    """The norms take them, as the norms of 16-bit outputs do; the others refuse them."""
    from roost_b200.kernels.library import KernelError
    x, w = rand((2, 3, 96), torch.bfloat16, 1), rand((96,), torch.bfloat16, 2)
    for call in (lambda v: kernels.rms_norm_e4m3(v, w, 1e-6), lambda v: kernels.add_rms_norm_e4m3(v, torch.ones_like(v), w, 1e-6)):
        (q, scale), (flat, flat_scale) = call(x), call(x.reshape(6, 96))
        assert q.shape[:-1] == scale.shape == (2, 3)
        assert torch.equal(q.reshape(6, -1).view(torch.uint8), flat.view(torch.uint8)) and torch.equal(scale.reshape(6), flat_scale)
    for call in (kernels.quantise_e4m3, kernels.silu_mul_e4m3):
        with pytest.raises(KernelError):
            call(x)


def test_no_rows(kernels):
    x = torch.empty((0, 256), dtype=torch.bfloat16, device="cuda")
    w = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    for q, scale in (kernels.quantise_e4m3(x), kernels.rms_norm_e4m3(x, w, 1e-6), kernels.add_rms_norm_e4m3(x, x.clone(), w, 1e-6)):
        assert q.shape == (0, 256) and scale.shape == (0,)
    assert kernels.silu_mul_e4m3(x)[0].shape == (0, 128)
    wq, ws = kernels.quantise_e4m3(rand((64, 256), torch.float32, 1))
    assert kernels.gemm_e4m3(q, scale, wq, ws).shape == (0, 64)


def test_refusals(kernels):
    from roost_b200.kernels.library import KernelError
    x = rand((4, 64), torch.bfloat16, 1)
    q, s = kernels.quantise_e4m3(x)
    w = torch.ones(64, device="cuda")
    bad = [lambda: kernels.quantise_e4m3(x.half()), lambda: kernels.quantise_e4m3(x.t()), lambda: kernels.quantise_e4m3(x.cpu()),
           lambda: kernels.quantise_e4m3(torch.empty((1, 60000), device="cuda")),
           lambda: kernels.silu_mul_e4m3(x[:, :63].contiguous()), lambda: kernels.silu_mul_e4m3(x, 12),
           lambda: kernels.rms_norm_e4m3(x, w[:32], 1e-6), lambda: kernels.rms_norm_e4m3(x, w, 0.0), lambda: kernels.rms_norm_e4m3(x, w.half(), 1e-6),
           lambda: kernels.add_rms_norm_e4m3(x, x[:2].contiguous(), w, 1e-6),
           lambda: kernels.add_rms_norm_e4m3(x.float(), x.clone(), w, 1e-6),
           lambda: kernels.rms_norm_e4m3(x, w, 1e-6, torch.zeros(2, dtype=torch.int64, device="cuda")),
           lambda: kernels.gemm_e4m3(q, s, q[:, :32], s), lambda: kernels.gemm_e4m3(q, s[:2], q, s), lambda: kernels.gemm_e4m3(q, s, q, s.double()),
           lambda: kernels.gemm_e4m3(x, s, q, s), lambda: kernels.gemm_e4m3(q, s, q, s, torch.float16)]
    for call in bad:
        with pytest.raises(KernelError):
            call()


def test_a_layers_products_in_one_graph(kernels):
    """Norm, product, gate, product as a layer uses them, captured once and replayed on new inputs: the same bits as the calls."""
    H, I, T = 512, 1024, 24
    gate_up, gs = kernels.quantise_e4m3(rand((2 * I, H), torch.float32, 1, 0.04))
    down, ds = kernels.quantise_e4m3(rand((H, I), torch.float32, 2, 0.04))
    w = torch.ones(H, dtype=torch.bfloat16, device="cuda")
    x, res = rand((T, H), torch.bfloat16, 3), rand((T, H), torch.bfloat16, 4)

    def layer(x, res):
        q, s = kernels.add_rms_norm_e4m3(x, res, w, 1e-6)
        q, s = kernels.silu_mul_e4m3(kernels.gemm_e4m3(q, s, gate_up, gs), 0)
        return kernels.gemm_e4m3(q, s, down, ds)

    xs, rs = x.clone(), res.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(xs, rs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(xs, rs)
    for seed in (5, 6):
        x2, r2 = rand((T, H), torch.bfloat16, seed), rand((T, H), torch.bfloat16, seed + 10)
        xs.copy_(x2), rs.copy_(r2)
        graph.replay()
        want = layer(x2, r2)
        assert torch.equal(y, want) and torch.equal(rs, r2)
