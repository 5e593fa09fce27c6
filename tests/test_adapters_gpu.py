"""Low-rank adapters of many requests beside a shared projection, against the formula in float64."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24      # float32: half a step, relative to the value


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def want_and_bound(y, x, a, b, scale, counts, slots, widths, ranks, h_half):
    """y after the adapters in float64, and how far a 32-bit sum may be: a step for each of the additions (the tensor cores cut off) of sums no
    larger than those of the magnitudes, ``h_half`` for what h is rounded to between the products, a half step for the scale and the last sum, and
    the output's rounding."""
    y64, bound = y.double().clone(), torch.zeros_like(y, dtype=torch.float64)
    K, at = x.shape[1], 0
    for n, s in zip(counts, slots):
        if s >= 0:
            rank, lo = int(ranks[s]) if ranks is not None else a.shape[2], 0
            for p, width in enumerate(widths):
                xa, aa, bb = x[at:at + n].double(), a[s, p, :rank].double(), b[s, lo:lo + width, :rank].double() * float(scale[s])
                delta = (xa @ aa.t()) @ bb.t()
                most = (xa.abs() @ aa.abs().t()) @ bb.abs().t()
                y64[at:at + n, lo:lo + width] += delta
                here = y64[at:at + n, lo:lo + width].abs()
                bound[at:at + n, lo:lo + width] = ((K + rank + 4) * 2 * HALF + h_half) * most + (torch.finfo(y.dtype).eps / 2 + HALF) * here
                lo += width
        at += n
    return y64, bound


def case(kernels, dtype, out, counts, slots, S, R, K, widths, ranks=None, pad=0, seed=1, spare=0):
    T, N, P = sum(counts) + spare, sum(widths), len(widths)
    x = rand((T, K + pad), dtype, seed)[:, pad:]
    y = rand((T, N + pad), out, seed + 1)[:, pad:]
    a, b = rand((S, P, R, K), dtype, seed + 2, K ** -0.5), rand((S, N, R), dtype, seed + 3, 0.5)
    scale = 0.5 + torch.rand(S, generator=torch.Generator().manual_seed(seed + 4)).cuda()
    if ranks is not None:
        ranks = torch.tensor(ranks, dtype=torch.int32).cuda()
        for s in range(S):     # what lies behind a slot's rank is not used, whatever it holds
            r = min(max(int(ranks[s]), 0), R)
            a[s, :, r:] = float("nan")
            b[s, :, r:] = float("inf")
    plan = kernels.adapter_plan(counts, slots)
    clamped = None if ranks is None else ranks.clamp(0, R)
    a0, b0 = torch.nan_to_num(a, nan=0.0), torch.nan_to_num(b, posinf=0.0)
    # h enters the second product as two bfloat16 numbers (2^-17 of it is left out), or three where the output is float32, or as it is
    want, bound = want_and_bound(y, x, a0, b0, scale, counts, slots, widths, clamped, 2.0 ** -17 if out == torch.bfloat16 else 2 * HALF)
    before = y.clone()
    got = kernels.adapters_add_(y, x, a, b, scale, plan, widths=widths, ranks=ranks)
    assert got is y
    worst = float(((y.double() - want).abs() / bound.clamp_min(1e-300)).max()) if y.numel() else 0.0
    still = bound == 0
    assert torch.equal(y[still], before[still]), "rows without an adapter stay as they are"
    print(f"MEASURED adapters {len(counts)} requests, {T} tokens: {worst:.3f} of the bound")
    assert worst <= 1.0
    y2 = before.clone()
    kernels.adapters_add_(y2, x, a, b, scale, plan, widths=widths, ranks=ranks)
    assert torch.equal(y, y2), "the same bits on every run"
    return y


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)]


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("counts,slots", [([1], [0]), ([1, 1, 1], [2, -1, 2]), ([1] * 40, [i % 3 for i in range(40)]), ([17], [1]), ([64], [1]), ([65, 3], [0, 1]),
                                          ([200, 1, 0, 129, 5], [1, 2, 0, 1, -1]), ([3, 0, 2], [-1, -1, -1])])
@pytest.mark.parametrize("R,K,widths", [(8, 64, (64,)), (16, 1000, (256, 64, 72)), (64, 512, (200, 200)), (5, 77, (33, 1)), (128, 256, (130,))])
def test_sizes(kernels, dtype, out, counts, slots, R, K, widths):
    case(kernels, dtype, out, counts, slots, 3, R, K, widths)


@pytest.mark.parametrize("dtype,out", TYPES)
def test_ranks_of_slots(kernels, dtype, out):
    ranks = [0, 1, 7, 8, 9, 24, 32, 40, -3]
    case(kernels, dtype, out, [4] * 9 + [70, 30], list(range(9)) + [2, 4], 9, 32, 264, (128, 40, 48), ranks=ranks)
    case(kernels, dtype, out, [1] * 9, list(range(9)), 9, 32, 264, (128, 40, 48), ranks=ranks)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("pad", [8, 3])
def test_rows_that_lie_apart(kernels, dtype, out, pad):
    case(kernels, dtype, out, [5, 80, 1], [1, 0, 1], 2, 16, 320, (96, 32), pad=pad)


def test_rows_behind_the_last_request(kernels):
    case(kernels, torch.bfloat16, torch.bfloat16, [5, 20], [0, 1], 2, 16, 256, (128,), spare=9)


@pytest.mark.parametrize("dtype,out", TYPES)
def test_larger_sizes(kernels, dtype, out):
    case(kernels, dtype, out, [1] * 20, [i * 5 % 16 for i in range(20)], 16, 16, 4096, (4096, 1024, 1024))
    case(kernels, dtype, out, [300, 211, 2], [3, 0, 2], 4, 32, 2048, (2048, 2048))


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("R,K,widths", [(64, 4096, (2048, 512, 512)), (128, 4104, (1000, 264, 8, 256)), (512, 2056, (640,)), (72, 8200, (96, 5000)), (24, 8, (256,)),
                                        (64, 1024, (8,) * 8)])
def test_large_ranks(kernels, dtype, out, R, K, widths):
    """h is up to 512 numbers a token: few tokens and tiles of 64, ranks that end inside a block of 32, one block of the inputs and many."""
    ranks = [R, R - 7, 1, 40 if R > 40 else 9]
    case(kernels, dtype, out, [1, 3, 1, 2, 1], [0, 1, 2, -1, 3], 4, R, K, widths)
    case(kernels, dtype, out, [1, 3, 1, 2, 1], [0, 1, 2, -1, 3], 4, R, K, widths, ranks=ranks)
    case(kernels, dtype, out, [70, 1, 64, 90], [1, 2, 3, 0], 4, R, K, widths, ranks=ranks)


def test_offsets_beyond_32_bits(kernels):
    """Rows of y and of b that lie more than 2 ** 31 numbers behind the first."""
    T, N, R, K, S = 40000, 60000, 8, 64, 5000
    y = torch.zeros((T, N), dtype=torch.bfloat16, device="cuda")
    x = rand((T, K), torch.bfloat16, 1)
    a = rand((S, 1, R, K), torch.bfloat16, 2)
    b = torch.zeros((S, N, R), dtype=torch.bfloat16, device="cuda")
    b[-1] = rand((N, R), torch.bfloat16, 3)
    scale = torch.full((S,), 0.5, device="cuda")
    kernels.adapters_add_(y, x, a, b, scale, kernels.adapter_plan([T - 5, 5], [-1, S - 1]))
    want, bound = want_and_bound(torch.zeros_like(y[-5:]), x[-5:], a[-1:], b[-1:], scale[:1], [5], [0], (N,), None, 2.0 ** -17)
    assert bool(((y[-5:].double() - want).abs() <= bound).all()) and not bool(y[:-5].any())


def test_a_list_that_is_wrong_reaches_nothing(kernels):
    """Slots that do not exist and tokens outside the step are passed over."""
    from roost_b200.kernels.library import AdapterPlan
    x, y = rand((4, 64), torch.bfloat16, 1), rand((4, 64), torch.bfloat16, 2)
    a, b, scale = rand((2, 1, 8, 64), torch.bfloat16, 3), rand((2, 64, 8), torch.bfloat16, 4), torch.ones(2, device="cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32).cuda()
    before = y.clone()
    kernels.adapters_add_(y, x, a, b, scale, AdapterPlan(ints([9, -1, 3]), ints([[0, 0, 2], [2, 2, 3], [-1, 2, 3], [1, 3, 9], [1, 2, 2]]), 4))
    assert torch.equal(y, before)
    kernels.adapters_add_(y, x, a, b, scale, AdapterPlan(ints([9, -1, 3]), ints([[1, -5, 7]]), 4))
    assert torch.equal(y[:3], before[:3]) and not torch.equal(y[3], before[3])


def test_a_rows_nan_stays_in_its_row(kernels):
    x, y = rand((70, 256), torch.bfloat16, 1), rand((70, 128), torch.bfloat16, 2)
    a, b, scale = rand((1, 1, 16, 256), torch.bfloat16, 3), rand((1, 128, 16), torch.bfloat16, 4), torch.ones(1, device="cuda")
    plan = kernels.adapter_plan([70], [0])
    clean = kernels.adapters_add_(y.clone(), x, a, b, scale, plan)
    x[9, 200] = float("nan")
    x[33, 0] = float("inf")
    got = kernels.adapters_add_(y.clone(), x, a, b, scale, plan)
    assert torch.isnan(got[9]).all() and not torch.isfinite(got[33]).any()
    keep = [i for i in range(70) if i not in (9, 33)]
    assert torch.equal(got[keep], clean[keep])


def test_on_another_stream_and_in_a_graph(kernels):
    x, y = rand((30, 512), torch.bfloat16, 1), rand((30, 256), torch.bfloat16, 2)
    a, b, scale = rand((4, 1, 16, 512), torch.bfloat16, 3, 0.05), rand((4, 256, 16), torch.bfloat16, 4), torch.ones(4, device="cuda")
    plan = kernels.adapter_plan([1] * 30, [i % 4 for i in range(30)])
    want = kernels.adapters_add_(y.clone(), x, a, b, scale, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.adapters_add_(y.clone(), x, a, b, scale, plan)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    static = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.adapters_add_(static, x, a, b, scale, plan)
    for _ in range(2):
        static.copy_(y)
        graph.replay()
        assert torch.equal(static, want)


def test_refusals(kernels):
    from roost_b200.kernels.library import KernelError
    x, y = rand((4, 64), torch.bfloat16, 1), rand((4, 96), torch.bfloat16, 2)
    a, b, scale = rand((2, 1, 8, 64), torch.bfloat16, 3), rand((2, 96, 8), torch.bfloat16, 4), torch.ones(2, device="cuda")
    plan, ranks = kernels.adapter_plan([2, 2], [0, 1]), torch.zeros(2, dtype=torch.int32, device="cuda")
    ok = dict(y=y, x=x, a=a, b=b, scale=scale, plan=plan)
    wide = rand((2, 1, 520, 64), torch.bfloat16, 3)
    for change in (dict(y=x, b=rand((2, 64, 8), torch.bfloat16, 4)), dict(x=x[:3]), dict(x=x.float()), dict(a=a[:, :, :, :32].contiguous()), dict(b=b[:1]), dict(b=b.float()), dict(scale=scale.double()), dict(scale=scale[:1]),
                   dict(widths=(64, 32)), dict(widths=(95,)), dict(ranks=ranks[:1]), dict(ranks=ranks.long()), dict(y=y.cpu()), dict(y=y.half()),
                   dict(plan=kernels.adapter_plan([9], [0])), dict(a=wide, b=rand((2, 96, 520), torch.bfloat16, 1))):
        with pytest.raises(KernelError):
            kernels.adapters_add_(**{**ok, **change})


def test_norm_product_and_adapters_of_a_layer(kernels):
    """The run as a layer uses it: the norm's rows in 8 bits and beside them the norm itself, which the adapters read; the product; the adapters on
    what it made. Against the formulas in float64, with the rounding of every step between them."""
    T, H, widths, S, R = 37, 512, (512, 128, 128), 3, 16
    counts, slots = [1] * 5 + [20, 12], [0, 1, 2, -1, 0, 1, -1]
    x, res = rand((T, H), torch.bfloat16, 1), rand((T, H), torch.bfloat16, 2)
    norm_w = rand((H,), torch.bfloat16, 3, 0.1) + 1
    w, w_scale = kernels.quantise_e4m3(rand((sum(widths), H), torch.float32, 4, 0.04))
    a, b, scale = rand((S, 3, R, H), torch.bfloat16, 5, 0.04), rand((S, sum(widths), R), torch.bfloat16, 6, 0.3), torch.ones(S, device="cuda")
    plan = kernels.adapter_plan(counts, slots)
    q, q_scale, kept = kernels.add_rms_norm_e4m3(x, res, norm_w, 1e-6, keep=True)
    y = kernels.gemm_e4m3(q, q_scale, w, w_scale)
    base = y.clone()
    kernels.adapters_add_(y, kept, a, b, scale, plan, widths=widths)
    want, bound = want_and_bound(base, kept, a, b, scale, counts, slots, widths, None, 2.0 ** -17)
    assert bool(((y.double() - want).abs() <= bound).all())
    s = res.double()
    v = s / torch.sqrt(s.square().mean(-1, keepdim=True) + 1e-6) * norm_w.double()
    rows = (q.double() * q_scale.double()[:, None])
    assert float(((rows - v).abs() - 2.0 ** -4 * v.abs() - 2.0 ** -10 * q_scale.double()[:, None] - 1e-5 * v.abs()).max()) <= 0      # e4m3: half a step, 2^-10 below 2^-6
    exact = rows @ (w.double() * w_scale.double()[:, None]).t()
    most = rows.abs() @ (w.double().abs() * w_scale.double()[:, None]).t()
    assert bool(((base.double() - exact).abs() <= (2.0 ** -8 + 3 * HALF) * exact.abs() + H * 2 * HALF * most).all())
