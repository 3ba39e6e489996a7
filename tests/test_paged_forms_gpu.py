"""Forms of the paged operators beside those of test_paged_gpu.py: rotated widths and head layouts
of append, batches that are mostly idle, tables wider than any sequence."""
import pytest
import torch

from test_paged_gpu import BF, H, HD, U, Pool, append_ref, close, decode_ref, gen, i32, normal, run_decode
from vx27_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rope_dim", [0, 16, 48, 128, 256])
@pytest.mark.parametrize("nq,nkv,n", [(5, 1, 3), (8, 8, 1), (1, 1, 40), (7, 1, 2000)])
def test_append_rotated_dims_and_heads(cuda, rope_dim, nq, nkv, n):
    """24 fp32 roundings in all, relative to the larger of a rotated pair, and the bf16 one of K."""
    g = gen(60)
    rope = ops.rope_table(4096, rope_dim) if rope_dim else torch.empty(4096, 0, device="cuda")
    pool = Pool(g, [100 + n], nkv, 16)
    x, kv, vv = normal(g, n, nq, HD), normal(g, n, nkv, HD), normal(g, n, nkv, HD)
    qw, kw = (1 + 0.1 * normal(g, HD) for _ in range(2))
    slots = torch.arange(100, 100 + n, dtype=torch.int32, device="cuda")
    pos = slots + 1000
    q = torch.empty_like(x)
    ops.gqa_paged_append(x, kv, vv, qw, kw, rope, pos, slots, pool.table, pool.k, pool.v, q,
                         seq=torch.zeros_like(slots))
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    page, row = pool.where(0, slots)
    for got, src, w, h in ((q, x, qw, 0), (pool.k[page, :, row], kv, kw, H)):
        ref = append_ref(src, w, False, rope, pos)
        size = ref.abs()
        r = rope_dim // 2
        if r:
            size[..., :2 * r] = (ref[..., :r].square() + ref[..., r:2 * r].square()).sqrt().repeat(1, 1, 2)
        close(got, ref, 24 * U * size + h * ref.abs())
    assert torch.equal(pool.v[page, :, row], vv.to(BF))


@pytest.mark.parametrize("n", [1, 900, 9000])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4)])
def test_decode_one_live_lane_among_idle_ones(cuda, n, weights, window, sinks):
    """64 lanes, one of them with a sequence, in tables four times as wide as it needs."""
    g = gen(61)
    B, at, nkv = 64, 37, 2
    lens = [0] * B
    lens[at] = n
    pool = Pool(g, lens, nkv, 64, max_pages=4 * ((n + 63) // 64))
    q, gate = normal(g, B, 12, HD), normal(g, B, 12, HD)
    w = normal(g, B, nkv, pool.max_pages * 64).abs() if weights else None
    before = w.clone() if weights else None
    got = run_decode(pool, q, gate, lens, torch.float32, window, sinks, w)
    ref, tol, sums, stol = decode_ref(pool, q, gate, lens, window, sinks, False, True)
    close(got, ref, tol)
    assert (got[torch.tensor(lens) == 0] == 0).all()
    if weights:
        close(w, before.double() + sums, stol + 2 * U * (before.double() + sums))
        assert torch.equal(w[sums == 0], before[sums == 0])


@pytest.mark.parametrize("nkv,G", [(1, 6), (2, 4), (8, 1)])
def test_decode_long_sequence_of_few_heads(cuda, nkv, G):
    """Items that every run shares: as many records as there are runs, over the heads."""
    g = gen(62)
    pool = Pool(g, [40_000], nkv, 128)
    q = normal(g, 1, nkv * G, HD)
    for out in (torch.float32, BF):
        got = run_decode(pool, q, None, [40_000], out)
        ref, tol, _, _ = decode_ref(pool, q, None, [40_000], 0, 0, out == BF, out != BF)
        close(got, ref, tol)
