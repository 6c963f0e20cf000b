"""`expert_plan` over millions of pairs: the same stable sort, in time that grows with the pairs."""

import pytest
import torch

import opengemm_b200 as og

pytestmark = pytest.mark.gpu


def check(pairs, top_k, experts, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    indices = torch.randint(-1, experts + 1, (pairs // top_k, top_k), generator=g, device="cuda", dtype=torch.int32)
    plan = og.expert_plan(indices, experts)
    flat = indices.flatten()
    valid = (flat >= 0) & (flat < experts)
    counts = torch.bincount(flat[valid], minlength=experts)
    assert plan.offsets[0] == 0 and torch.equal(plan.offsets[1:].long(), counts.cumsum(0))
    order = torch.where(valid, flat, experts).sort(stable=True).indices[: int(plan.offsets[-1])]
    assert torch.equal(plan.tokens[: order.numel()].long(), order // top_k)
    positions = torch.full((flat.numel(),), -1, device="cuda", dtype=torch.int32)
    positions[order] = torch.arange(order.numel(), device="cuda", dtype=torch.int32)
    assert torch.equal(plan.positions.flatten(), positions)


@pytest.mark.parametrize("pairs,top_k,experts", [(8192 * 31 + 5, 1, 3), (8192 * 32, 8, 64), (8192 * 33 - 8, 8, 1000), (8192 * 64 + 1, 1, 1024),
                                                 (8192 * 129 - 3, 1, 1), (8192 * 700 + 40, 8, 33), (8192 * 2049 + 2, 2, 128)])
def test_plan_of_many_chunks_is_a_stable_sort(pairs, top_k, experts):
    check(pairs, top_k, experts)


def test_time_grows_with_the_pairs():
    """Eight times the pairs take about eight times as long, not sixty-four."""
    def milliseconds(pairs):
        indices = torch.randint(0, 512, (pairs // 8, 8), device="cuda", dtype=torch.int32)
        og.expert_plan(indices, 512)
        best = float("inf")
        for _ in range(3):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            og.expert_plan(indices, 512)
            end.record()
            end.synchronize()
            best = min(best, start.elapsed_time(end))
        return best

    assert milliseconds(2**26) < 20 * milliseconds(2**23)
