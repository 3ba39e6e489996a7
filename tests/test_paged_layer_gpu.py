"""GQALayer over a PagedKV: rounds that a server makes, against the same tokens one by one."""
import pytest
import torch

from test_paged_gpu import gen, gqa_layer, normal
from vx27_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("step_first", [True, False])
@pytest.mark.parametrize("captured", [False, True])
def test_a_prompt_of_one_token_beside_steps(cuda, step_first, captured):
    """Sequence 0 decodes while sequence 1's prompt ends in a piece of one token: in one round
    both give what they give in rounds of their own, whichever call comes first, and the prompt
    adds nothing to the sums."""
    from vx27_b200.paged import PagedKV
    layer, B, H = gqa_layer(50), 2, 512
    g = gen(51)
    x0, x1, x, xp = normal(g, 20, H), normal(g, 30, H), normal(g, B, H), normal(g, 1, H)
    caches = [PagedKV(1, B, 12, 4, 16, 2, weights=True) for _ in range(2)]
    ws = [c.workspace(12) for c in caches]
    for c, w in zip(caches, ws):
        c.k.zero_()
        c.v.zero_()
        at = c.extend({0: 20, 1: 30})
        layer.prompt_paged(x0, c, 0, 0, *at[0], w)
        layer.prompt_paged(x1, c, 0, 1, *at[1], w)
    graph = torch.cuda.CUDAGraph()
    if captured:
        layer.step_paged(x, caches[0], 0, ws[0])  # all lanes idle
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y = layer.step_paged(x, caches[0], 0, ws[0])

    def step():
        if captured:
            graph.replay()
            return y
        return layer.step_paged(x, caches[0], 0, ws[0])
    at = caches[0].extend({0: 1, 1: 1}, prompts=[1])
    if step_first:
        got = step()
    got_p = layer.prompt_paged(xp, caches[0], 0, 1, *at[1], ws[0])
    if not step_first:
        got = step()
    c, w = caches[1], ws[1]
    ref_p = layer.prompt_paged(xp, c, 0, 1, *c.extend({1: 1}, prompts=[1])[1], w)
    c.extend({0: 1})
    ref = layer.step_paged(x, c, 0, w)
    assert torch.equal(got[0], ref[0]) and torch.equal(got_p, ref_p)
    assert (got[1] == 0).all() and (c.sums[0, 1] == 0).all()
    for i, s in ((0, 21), (1, 31)):
        assert caches[0].length(i) == c.length(i) == s
    for name in ("k", "v"):  # the pages may be others
        a, b = (torch.stack([getattr(m, name)[0][m.table[i].long().clamp_min(0)] *
                             (m.table[i] >= 0)[:, None, None, None] for i in range(B)]) for m in caches)
        assert torch.equal(a, b)
    assert torch.equal(caches[0].sums, c.sums)
    assert ops.device_status() == 0
