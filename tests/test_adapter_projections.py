"""An adapter that names some of a model's projections touches those and no others; room is kept where an adapter can be loaded."""
import pytest
import torch

from roost_b200.engine.model import load_model
from tests.fake_kernels import FakeKernels
from tests.helpers import random_ids
from tests.test_adapter_models import write_adapter


class Recording(FakeKernels):
    """Keeps what every call of the adapters would add to."""

    def __init__(self):
        self.calls = []

    def adapters_add_(self, y, x, a, b, scale, plan, widths=None, ranks=None):
        self.calls.append((tuple(widths), [int(ranks[int(slot)]) for slot in plan.tiles[:, 0] if int(slot) >= 0]))
        return super().adapters_add_(y, x, a, b, scale, plan, widths, ranks)


def test_ranks_are_a_projections_own(tiny_model_dirs, tmp_path):
    """The queries' adapter alone: the products of the attention's output and of the feed-forward have nothing to add, and after a reload they do."""
    base = tiny_model_dirs["A"]
    write_adapter(tmp_path / "q", base, 4, 8.0, 1, ("self_attn.q_proj",))
    write_adapter(tmp_path / "all", base, 6, 6.0, 2)
    kernels = Recording()
    model = load_model(base, torch.float32, "cpu", kernels, adapters=(2, 8))
    model.load_adapter("q", tmp_path / "q")
    model.load_adapter("all", tmp_path / "all")
    for block in model.blocks:
        assert block.mixer.qkv.adapters.ranks.tolist() == [4, 6]
        for other in (block.mixer.out, block.feed_forward.gate_up, block.feed_forward.down):
            assert other.adapters.ranks.tolist() == [0, 6]
    assert model.rt.adapters.ranks.tolist() == [4, 6]

    from roost_b200.engine.executor import StepEntry, StepExecutor
    ex = StepExecutor(model, max_tokens=64)
    ex.adapter_of["a"] = model.rt.adapters.names["q"]
    ex.step([StepEntry("a", random_ids(5, 130, 1), [0])])
    ranks = [r for _, r in kernels.calls]
    assert len(ranks) == 4 * len(model.blocks) and all(set(r) == {4} for r in ranks[0::4]) and all(set(r) == {0} for i, r in enumerate(ranks) if i % 4)

    model.load_adapter("q", tmp_path / "all")
    assert all(p.adapters.ranks.tolist() == [6, 6] for b in model.blocks for p in (b.mixer.qkv, b.mixer.out, b.feed_forward.gate_up, b.feed_forward.down))


@pytest.mark.gpu
def test_rows_of_a_projection_that_is_not_named_keep_their_bits(kernels, tiny_model_dirs, tmp_path):
    base = tiny_model_dirs["D"]
    write_adapter(tmp_path / "q", base, 4, 8.0, 1, ("self_attn.q_proj",))
    model = load_model(base, torch.bfloat16, "cuda", kernels, adapters=(2, 8))
    slot = model.load_adapter("q", tmp_path / "q")
    for proj, touched in ((model.blocks[0].mixer.qkv, True), (model.blocks[0].mixer.out, False), (model.blocks[0].feed_forward.down, False)):
        y = torch.full((9, proj.out_features), -0.0, dtype=torch.bfloat16, device="cuda")
        x = torch.randn((9, proj.in_features), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
        proj.adapters.add_(y, x, kernels.adapter_plan([9], [slot]))
        assert bool(torch.signbit(y).all() and not y.any()) != touched
