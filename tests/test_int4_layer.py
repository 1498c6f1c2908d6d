"""``Int4Experts`` in the places an ``ExpertContext`` has: the refusals and exchanges that they share."""
import pytest
import torch

gpu = pytest.mark.gpu


class Context:
    """What ``Int4Experts`` asks of its own context, without a device."""

    device = torch.device("cpu")

    def _check_x(self, x):
        return x


def experts_without_a_device():
    from constellation_b200.int4 import Int4Experts

    ex = object.__new__(Int4Experts)
    ex._ctx, ex.device, ex._shared = Context(), Context.device, None
    ex._routed = lambda x, idx, weight, extra, dtype: ("routed", extra)
    return ex


def test_a_shared_expert_that_is_not_resident_is_an_error():
    """As with ``ExpertContext``: an empty range needs no shared expert, any other does."""
    ex = experts_without_a_device()
    x, idx, weight = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    for b, e in ((0, 0), (2, 2), (4, 4)):
        assert ex.moe_routed_range(x, idx, weight, b, e) == ("routed", None)
    for b, e in ((0, 4), (1, 2), (3, 4)):
        with pytest.raises(RuntimeError, match="no shared expert is resident"):
            ex.moe_routed_range(x, idx, weight, b, e)
    with pytest.raises(RuntimeError, match="no shared expert is resident"):
        ex.moe_routed(x, idx, weight, add_shared=True)


def test_an_exchange_that_a_compute_object_does_not_know_is_refused_at_once():
    from constellation_b200.ep import ExpertParallelMoE
    from constellation_b200.stack import MoEStack, StackLayer

    ex = experts_without_a_device()
    for mode in ("p2p", "alltoall"):
        with pytest.raises(ValueError, match="Int4Experts"):
            ExpertParallelMoE(ex, rank=0, world=2, n_routed_experts=4, mode=mode)
        with pytest.raises(ValueError, match=mode):
            MoEStack([StackLayer(ex, None, None)], rank=1, world=2, n_routed_experts=4, mode=mode)
        assert ExpertParallelMoE(ex, rank=0, world=1, n_routed_experts=4, mode=mode).c is ex  # nothing is exchanged
    assert ExpertParallelMoE(ex, rank=1, world=2, n_routed_experts=4).c is ex
