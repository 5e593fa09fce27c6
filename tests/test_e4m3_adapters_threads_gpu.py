"""The 8-bit row kernels and the adapters called by several host threads at once, each on a stream of its own."""
import threading

import pytest
import torch

from tests.test_e4m3_gpu import rand

pytestmark = pytest.mark.gpu


def together(calls, times):
    """Every call ``times`` times in a thread and on a stream of its own, all at once; what each thread raised."""
    errors, start = [], threading.Barrier(len(calls))

    def loop(call):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(60)
                for _ in range(times):
                    call()
        except Exception as e:      # noqa: BLE001: any of them is the test's failure
            errors.append(e)

    threads = [threading.Thread(target=loop, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return errors


@pytest.mark.parametrize("kind", ["quantise", "silu_mul", "norm"])
def test_rows_of_different_lengths(kernels, kind):
    """Odd rows stand in shared memory, as much as the row is long: a short row's call does not take a long one's room."""
    def call(cols):
        x = rand((1, 2 * cols if kind == "silu_mul" else cols), torch.bfloat16, cols)
        w = torch.ones(cols, device="cuda")
        return {"quantise": lambda: kernels.quantise_e4m3(x), "silu_mul": lambda: kernels.silu_mul_e4m3(x), "norm": lambda: kernels.rms_norm_e4m3(x, w, 1e-6)}[kind]

    assert not together([call(51167), call(10307), call(51165), call(20001)], 1500)


def test_adapters_of_different_ranks(kernels):
    def call(rank, tokens):
        x, y = rand((tokens, 64), torch.float32, 1), torch.zeros((tokens, 32), device="cuda")
        a, b, scale = rand((1, 1, rank, 64), torch.float32, 2), rand((1, 32, rank), torch.float32, 3), torch.ones(1, device="cuda")
        plan = kernels.adapter_plan([tokens], [0])
        return lambda: kernels.adapters_add_(y, x, a, b, scale, plan)

    assert not together([call(512, 64 * 40), call(200, 64 * 40), call(500, 64 * 40), call(230, 64 * 40)], 1500)
