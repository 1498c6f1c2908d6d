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


class Exchange:
    """The collectives of ranks that are threads of this process; a group is the rank's number.  Every rank launches on the
    device's default stream, so what one has enqueued before the barrier is done before what another enqueues after."""

    from torch.distributed import ReduceOp

    def __init__(self, world):
        import threading

        self.world, self.slots, self.barrier = world, [None] * world, threading.Barrier(world, timeout=60)

    def _all(self, rank, t, use):
        self.slots[rank] = t
        self.barrier.wait()
        use(self.slots)
        self.barrier.wait()

    def all_gather_into_tensor(self, out, t, group):
        self._all(group, t, lambda every: out.copy_(torch.cat(every)))

    def reduce_scatter_tensor(self, out, t, op, group):
        assert op == self.ReduceOp.SUM
        self._all(group, t, lambda every: out.copy_(sum(every).chunk(self.world)[group]))


@gpu
@pytest.mark.parametrize("local_route_min", [1, 128])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_the_all_gather_exchange_over_int4_experts(monkeypatch, dt, local_route_min):
    """Two ranks with half of the experts each, against the layer in 64 bits with the same quantised weights."""
    from concurrent.futures import ThreadPoolExecutor

    from constellation_b200 import ep
    from constellation_b200.context import MoEConfig
    from constellation_b200.int4 import Int4Experts, quantize_int4

    world, Tl, E, H, I = 2, 9, 8, 256, 128
    cfg = MoEConfig(hidden_size=H, moe_intermediate_size=I, n_routed_experts=E, n_group=4, topk_group=2,
                    num_experts_per_tok=3)
    g = torch.Generator().manual_seed(11)
    ranks = [Int4Experts("cuda", cfg, max_tokens=world * Tl, n_local=E // world, first_expert=E // world * r)
             for r in range(world)]
    W = {}
    for e in [*range(E), -1]:
        parts = [quantize_int4((torch.randn(n, k, generator=g) * 0.05).cuda()) for n, k in ((2 * I, H), (H, I))]
        W[e] = [(torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1).double() - 8)
                * s.double().repeat_interleave(128, 1) for q, s, _ in parts]
        for r, ex in enumerate(ranks):
            if e < 0 or e // (E // world) == r:
                ex.load_expert(e, *parts)
    gate, bias = torch.randn(E, H, generator=g).cuda() * 0.1, torch.randn(E, generator=g).cuda() * 0.05
    x, residual = (torch.randn(world * Tl, H, generator=g).to("cuda", dt) for _ in range(2))
    exchange = Exchange(world)
    monkeypatch.setattr(ep, "dist", exchange)
    moe = [ep.ExpertParallelMoE(ex, rank=r, world=world, n_routed_experts=E, group=r, local_route_min=local_route_min)
           for r, ex in enumerate(ranks)]

    def forward(r):
        own = slice(r * Tl, (r + 1) * Tl)
        try:
            return moe[r].forward(x[own], gate, bias, residual=residual[own], out_dtype=torch.float32)
        except BaseException:
            exchange.barrier.abort()
            raise

    idx, weight = moe[0].routes(x, gate, bias)
    with ThreadPoolExecutor(world) as pool:
        out = torch.cat(list(pool.map(forward, range(world))))

    ref, slack = residual.double().clone(), torch.zeros(world * Tl, H, dtype=torch.float64, device="cuda")

    def add(t, e, factor):
        u = x[t].double() @ W[e][0].T
        h = u[:, I:] * torch.sigmoid(u[:, I:]) * u[:, :I]
        ref[t] += factor * (h @ W[e][1].T)
        slack[t] += factor.abs() * (h.abs() @ W[e][1].abs().T)

    add(torch.arange(world * Tl, device="cuda"), -1, torch.ones(world * Tl, 1, dtype=torch.float64, device="cuda"))
    for k in range(idx.shape[1]):
        for e in range(E):
            t = (idx[:, k] == e).nonzero().view(-1)
            add(t, e, weight[t, k, None].double())
    # the rows between the products are rounded, half a step of each; the fp32 sums add far less
    step = torch.finfo(dt).eps / 2
    assert ((out.double() - ref).abs() <= step * 1.05 * slack + 1e-6 * ref.abs() + 1e-6).all()
    for ex in ranks:
        ex.device_error()
