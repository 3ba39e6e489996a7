"""Prompt rows by themselves: what a row gets depends on the slots it sees, not on how many rows
are in the call, nor on what the other rows of its tile hold."""
import pytest
import torch

from test_paged_gpu import BF, HD, Pool, gen, normal, prompt_ref, run_prompt
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


def paged_prompt_error(T, s0, at, window=0, gate=True, nq=24, nkv=4):
    """Largest |error| over its bound of T rows with the same q after s0 slots, where the slots
    in `at` score 128, 256, ... (all heads) against about 4 at most elsewhere. The bound is
    prompt_ref's, whose score term grows with the scores' size."""
    g = gen(42)
    pool = Pool(g, [s0 + T], nkv, 64)
    q = normal(g, nkv, HD).to(BF)
    for i, slot in enumerate(at):
        page, row = pool.where(0, [slot])
        pool.k[page, :, row] = (q * (8 * (i + 1)))[None]
    q = q.repeat_interleave(nq // nkv, 0).expand(T, nq, HD).contiguous()
    gt = normal(g, T, nq, HD).to(BF) if gate else None
    got = run_prompt(pool, q, gt, s0, window, 4 if window else 0)
    ref, tol = prompt_ref(pool, q, gt, s0, window, 4 if window else 0)
    return float(((got.double() - ref).abs() / tol).max())


@pytest.mark.parametrize("T", [1, 64])
@pytest.mark.parametrize("s0,at,window", [
    (300, [200], 0),                            # one outlier, in the second tile of an uncut pair
    (700, [200, 500, 690], 0),                  # each further above the one before
    (700, [200, 500, 600], 300),                # behind the sinks' tile
    (20000, [1000, 7000, 13000, 19000], 0)])    # a pair that is cut into parts
def test_paged_maximum_that_leaves_all_before_it_behind(cuda, T, s0, at, window):
    """A key tile whose maximum is more than 2^126 times what came before: the sums of the
    earlier tiles are rescaled to nothing, as their weights underflow."""
    for gate in (True, False):
        assert paged_prompt_error(T, s0, at, window, gate) <= 1


def test_paged_maximum_odd_heads(cuda):
    """Pairs of two row tiles (an odd group of heads)."""
    for T, s0, at in ((1, 300, [200]), (300, 300, [200, 310, 450])):
        assert paged_prompt_error(T, s0, at, nq=5, nkv=1) <= 1


@pytest.mark.parametrize("cta_pairs", [True, False])
@pytest.mark.parametrize("act", [BF, torch.float32])
@pytest.mark.parametrize("T", [1, 64])
def test_contiguous_maximum_that_leaves_all_before_it_behind(cuda, T, act, cta_pairs):
    """The same for gqa_prefill. With norm weights of 3 and no rotation (cosines 1, sines 0), a
    key like q scores 9 * 256 / 16 = 144 and the others sqrt(81) = 9 sigma, so below 60 among a
    few hundred: the outlier's weight is 1 to within e^-80, and a row is its V row times the
    gate's sigmoid. Its weight, at most 2^8 (the maximum may lag by that), is rounded to bf16
    and its sum is not: 2^-8; the sigmoid 2^-20."""
    g = gen(43)
    p0, at, nq, nkv = 300, 200, 24, 4
    w = torch.full((HD,), 3.0, device="cuda")
    rope = torch.cat([torch.ones(512, 32, device="cuda"), torch.zeros(512, 32, device="cuda")], 1)
    q = normal(g, nkv, HD).to(act)
    k, v = (normal(g, p0 + T, nkv, HD).to(act) for _ in range(2))
    k[at] = q
    q = q.repeat_interleave(nq // nkv, 0)
    gate = normal(g, p0 + T, nq, HD).to(act)
    kc, vc = (torch.zeros(nkv, 512, HD, device="cuda", dtype=BF) for _ in range(2))
    out = torch.empty(p0 + T, nq, HD, device="cuda")
    for a, b in ((0, p0), (p0, p0 + T)):
        ops.gqa_prefill(q.expand(b - a, nq, HD).contiguous(), k[a:b], v[a:b], gate[a:b], w, w, rope,
                        kc, vc, out[a:b], p0=a, cta_pairs=cta_pairs)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    ref = v[at].to(BF).double().repeat_interleave(nq // nkv, 0) * torch.sigmoid(gate.double())
    err = (out.double() - ref).abs()[at:]  # of both calls' rows
    worst = float((err / ((2.0 ** -8 + 2.0 ** -18) * ref.abs()[at:] + 1e-30)).max())
    assert worst <= 1
