"""Results of the paged attention do not depend on what else is in the step:
sequences alone and in another order."""
import numpy as np
import pytest

from test_gpu_paged import Step

pytestmark = pytest.mark.gpu


def cuts(plan):
    """How a plan cuts each row block: (sequence, KV head, first row, rows) to
    the kernel and the runs of units of its items."""
    w, p = plan.words.cpu().numpy(), plan._c
    found = {}
    for kind, off, n in (("small", p.off_small, p.small_items), ("tile", p.off_tile, p.tile_items)):
        for seq, g, r0, rows, i0, i1, *_ in w[off:off + 12 * n].reshape(-1, 12).tolist():
            found.setdefault((seq, g, r0, rows), set()).add((kind, p.small_kind, i0, i1))
    return found


@pytest.mark.parametrize("values,cache,hd", [("f32", "bf16", 64), ("bf16", "bf16", 128), ("f32", "int8", 128), ("bf16", "int8", 64),
                                             ("f32", "f32", 64)])
def test_sequences_alone_and_in_another_order(values, cache, hd):
    import torch
    import llm_inference_edu_b200 as qb
    starts, counts, heads, kv = [900, 20, 0, 511, 2300], [1, 60, 200, 4, 1], 14, 2
    G = heads // kv
    s = Step(starts, counts, heads, kv, hd, values, cache, seed=4)
    whole = torch.from_numpy(s.attend())
    y, bound = (torch.from_numpy(x) for x in s.want())
    mine = cuts(s.plan)
    first = np.cumsum([0] + counts)
    alike = 0
    for order in [[i] for i in range(5)] + [[4, 3, 2, 1, 0], [2, 0, 4, 1, 3]]:
        rows = torch.cat([torch.arange(first[i], first[i + 1]) for i in order])
        plan = qb.PagedPlan(s.cache, s.tables[order], [starts[i] for i in order], [counts[i] for i in order], heads, dtype=values)
        out = torch.full((len(rows), heads, hd), 7.0, dtype=s.y.dtype, device="cuda")
        qb.paged_attention(s.q[rows.cuda()], s.cache, plan, out)
        got = torch.full_like(whole, float("nan"))
        got[rows] = out.double().cpu()
        assert ((got - y).abs() <= bound)[rows].all()
        for (seq, g, r0, n), how in cuts(plan).items():
            if mine.get((order[seq], g, r0, n)) != how:
                continue
            alike += 1
            for r in range(r0, r0 + n):
                t, h = first[order[seq]] + r // G, g * G + r % G
                assert torch.equal(got[t, h], whole[t, h]), (order, seq, g, r)
    assert alike
