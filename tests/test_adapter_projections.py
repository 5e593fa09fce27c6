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


def test_no_room_where_no_adapter_can_be_loaded(tiny_model_dirs, tmp_path):
    """A shared expert beside routed ones and the branches of a parallel mixer have no module that an adapter could name: they keep no room, a step with
    adapters runs nothing beside them, and a shared expert keeps the layout of its fused products."""
    import dataclasses

    from roost_b200.config.spec import ParallelMixerSpec, RoutedMlpSpec
    from roost_b200.engine.model import Model
    from roost_b200.parts import Runtime
    from roost_b200.parts.routed_mlp import RoutedMlp

    class Fused(FakeKernels):
        gemm_tcgen05_swiglu = None     # that the fused product exists is what chooses the layout

    spec = RoutedMlpSpec(hidden=64, experts=4, top=1, expert_intermediate=16, shared_intermediate=128)
    with_room = RoutedMlp(spec, Runtime(torch.bfloat16, "cpu", Fused(), adapters=(2, 8))).shared
    assert with_room.gate_up.adapters is None and with_room.down.adapters is None
    assert with_room.interleave == RoutedMlp(spec, Runtime(torch.bfloat16, "cpu", Fused())).shared.interleave == 128

    base = load_model(tiny_model_dirs["A"], torch.float32, "cpu", FakeKernels()).spec
    blocks = [dataclasses.replace(b, mixer=ParallelMixerSpec(hidden=64, branches=(b.mixer, b.mixer))) if i == 0 else b for i, b in enumerate(base.blocks)]
    names = {k: v for k, v in base.weight_names.items() if k != "blocks.0.mixer"}
    names["blocks.0.mixer"] = {f"{n}.{local}": t for n in range(2) for local, t in base.weight_names["blocks.0.mixer"].items()}
    model = Model(dataclasses.replace(base, blocks=blocks, weight_names=names), Runtime(torch.float32, "cpu", FakeKernels(), adapters=(2, 8)))
    branches = model.blocks[0].mixer.branches
    assert all(b.qkv.adapters is None and b.out.adapters is None for b in branches)
    loadable = {id(p) for p, _ in model.adapter_projections().values()}
    others = [model.blocks[0].feed_forward.gate_up, model.blocks[1].mixer.qkv, model.blocks[1].mixer.out, model.blocks[1].feed_forward.down]
    assert all(id(p.adapters) in loadable for p in others)
