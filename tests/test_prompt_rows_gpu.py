"""Prompt rows by themselves: what a row gets depends on the slots it sees, not on how many rows
are in the call, nor on what the other rows of its tile hold."""
import pytest
import torch

from test_paged_gpu import BF, HD, Pool, gen, normal
from vx27_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nq,nkv", [(24, 4), (5, 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_paged_rows_of_a_tile_that_is_not_full(cuda, nq, nkv, window, sinks):
    """T rows that end inside a warp, equal bit for bit to the same rows of 256: the slots that
    only later rows see have weight 0, and each row has sums and maxima of its own."""
    g = gen(40)
    s0, full = 40, 256
    pool = Pool(g, [s0 + full], nkv, 32)
    q, gate = normal(g, full, nq, HD).to(BF), normal(g, full, nq, HD).to(BF)
    ws = torch.empty(ops.gqa_paged_prefill_workspace_bytes(nkv, HD), dtype=torch.uint8, device="cuda")

    def run(T, gt):
        out = torch.full((T + 3, nq, HD), float("nan"), device="cuda", dtype=BF)
        ops.gqa_paged_prefill(q[:T], None if gt is None else gt[:T], pool.k, pool.v, pool.table[0],
                              out[:T], ws, s0=s0, window=window, sinks=sinks)
        torch.cuda.synchronize()
        assert ops.device_status() == 0
        assert out[T:].isnan().all()
        return out[:T]
    for gt in (gate, None):
        ref = run(full, gt)
        assert not ref.isnan().any()
        for T in (1, 31, 33, 97, 129, 250):
            assert torch.equal(run(T, gt), ref[:T]), T


@pytest.mark.parametrize("cta_pairs", [True, False])
@pytest.mark.parametrize("act,out_t", [(BF, BF), (BF, torch.float32), (torch.float32, torch.float32)])
def test_contiguous_rows_of_a_tile_that_is_not_full(cuda, cta_pairs, act, out_t):
    """The same for gqa_prefill, with its two kernels."""
    g = gen(41)
    p0, full, nq, nkv = 40, 256, 24, 4
    rope = ops.rope_table(512)
    w = torch.ones(HD, device="cuda")
    x = [normal(g, full, m, HD).to(act) for m in (nq, nkv, nkv, nq)]
    rows = normal(g, 2, nkv, 512, HD).to(BF)

    def run(T):
        kc, vc = rows[0].clone(), rows[1].clone()
        out = torch.full((T + 3, nq, HD), float("nan"), device="cuda", dtype=out_t)
        ops.gqa_prefill(*(t[:T] for t in x), w, w, rope, kc, vc, out[:T], p0=p0, cta_pairs=cta_pairs)
        torch.cuda.synchronize()
        assert ops.device_status() == 0
        assert out[T:].isnan().all()
        return out[:T]
    ref = run(full)
    assert not ref.isnan().any()
    for T in (1, 31, 33, 97, 129, 250):
        assert torch.equal(run(T), ref[:T]), T
