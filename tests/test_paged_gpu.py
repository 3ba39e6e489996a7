"""GQA over the paged cache against the formulas in 64 bits (torch, double, plain indexing).

Tolerances, with u = 2^-24 (fp32), h = 2^-8 (half a bf16 step, relative), w = the size of the
q.k terms, A_j = sum_d |q_d k_jd| / 16, and Av = sum_j p_j |v_j|:
* a score: 256 products summed in fp32 in any order are off by at most 256 u A; entering the
  tensor cores as two bf16 terms drops at most 2^-16 of each q (2^-24 as three): dS =
  (256 u + r) A, r = 2^-16 or 2^-24, with A at its largest over the row
* p_j = e^(s_j - m): relative error at most 2 dS (numerator and sum) + 16 u (exp2 and its
  argument's rounding) + r (its own terms); l likewise, so o is off by at most
  2 (2 dS + 16 u + r) Av + 256 u Av (the sum over slots, in tiles)
* prompts round p to bf16: h Av instead of r Av; q is bf16 as given, r = 0
* the gate's sigmoid: 8 u relative (2^-20 for the prompt's, by the SFU); a bf16 output h
"""
import numpy as np
import pytest
import torch

from vx27_b200 import ops

pytestmark = pytest.mark.gpu
HD = 256
U, H = 2.0 ** -24, 2.0 ** -8
BF = torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *s):
    return torch.randn(s, generator=g, device="cuda")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Pool:
    """Pages in random order; pages that no sequence owns and rows that nothing wrote are NaN."""

    def __init__(self, g, lens, nkv, ps, spare=3, max_pages=None):
        need = [(n + ps - 1) // ps for n in lens]
        self.ps, self.nkv = ps, nkv
        self.max_pages = max_pages or max(max(need), 1)
        n = sum(need) + spare
        self.k = torch.full((n, nkv, ps, HD), float("nan"), device="cuda", dtype=BF)
        self.v = self.k.clone()
        order = torch.randperm(n, generator=g, device="cuda").int()
        self.table = torch.full((len(lens), self.max_pages), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = order[at:at + m]
            at += m
        self.spare = order[at:]
        for b, m in enumerate(lens):
            self.write(b, 0, normal(g, m, nkv, HD).to(BF), normal(g, m, nkv, HD).to(BF))

    def where(self, b, slots):
        s = torch.as_tensor(slots, device="cuda").long()
        return self.table[b].long()[s // self.ps], s % self.ps

    def write(self, b, s0, k, v):
        if len(k):
            page, row = self.where(b, torch.arange(s0, s0 + len(k)))
            self.k[page, :, row], self.v[page, :, row] = k, v

    def rows(self, b, slots):
        """K and V [nkv][slots][256] in 64 bits."""
        page, row = self.where(b, slots)
        return (self.k[page, :, row].double().transpose(0, 1),
                self.v[page, :, row].double().transpose(0, 1))


def seen(n, window, sinks):
    lo = max(n - window, 0) if window else 0
    return [*range(min(sinks, lo)), *range(lo, n)]


def attend(q, k, v, mask=None):
    """q [nkv][rows][256], k, v [nkv][slots][256] -> (o, p, Av, max A) in 64 bits."""
    q = q.double()
    s = q @ k.mT / 16
    if mask is not None:
        s = s.masked_fill(~mask, float("-inf"))
    p = torch.softmax(s, -1)
    A = (q.abs() @ k.abs().mT / 16).amax(-1, keepdim=True)
    return p @ v, p, p @ v.abs(), A


def close(got, ref, tol):
    got = got.double()
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float((got - ref).abs().max()), float(tol.max()))


def decode_ref(pool, q, gate, lens, window, sinks, out_bf16, three):
    B, nq, nkv = q.shape[0], q.shape[1], pool.nkv
    r = 2.0 ** -24 if three else 2.0 ** -16
    ref, tol = torch.zeros(2, B, nq, HD, dtype=torch.float64, device="cuda")
    sums, stol = torch.zeros(2, B, nkv, pool.max_pages * pool.ps, dtype=torch.float64,
                             device="cuda")
    for b, n in enumerate(lens):
        slots = seen(n, window, sinks)
        if not slots:
            continue
        k, v = pool.rows(b, slots)
        o, p, av, A = attend(q[b].view(nkv, -1, HD), k, v)
        dp = 2 * (256 * U + r) * A + 16 * U + r
        ref[b], tol[b] = o.reshape(nq, HD), ((2 * dp + 256 * U) * av).reshape(nq, HD)
        at = torch.tensor(slots, device="cuda")
        sums[b][:, at] = p.sum(1)
        stol[b][:, at] = (2 * dp * p).sum(1)
    if gate is not None:
        s = torch.sigmoid(gate.double())
        ref, tol = ref * s, tol * s + 8 * U * (ref * s).abs()
    if out_bf16:
        tol = tol * (1 + H) + H * ref.abs()
    return ref, tol + 1e-30, sums, stol


def run_decode(pool, q, gate, lens, out_dtype, window=0, sinks=0, weights=None, n_parts=0,
               stream=None):
    B, nq = q.shape[:2]
    ws = torch.empty(ops.gqa_paged_workspace_bytes(B, nq, pool.nkv, HD, pool.max_pages * pool.ps,
                                                   window, sinks, weights is not None, n_parts),
                     dtype=torch.uint8, device="cuda")
    out = torch.full((B, nq, HD), float("nan"), device="cuda", dtype=out_dtype)
    ops.gqa_paged_decode(q, gate, pool.k, pool.v, pool.table, i32(lens), out, ws, window=window,
                         sinks=sinks, weight_sum=weights, n_parts=n_parts, stream=stream)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    return out


LENS = [0, 1, 15, 16, 17, 127, 128, 129, 300, 1000]


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("out", [torch.float32, BF])
@pytest.mark.parametrize("n_parts", [0, 1, 3, 7])
def test_decode_ragged(cuda, ps, out, n_parts):
    g = gen(1)
    pool = Pool(g, LENS, 4, ps)
    q, gate = normal(g, len(LENS), 24, HD), normal(g, len(LENS), 24, HD).to(BF)
    got = run_decode(pool, q, gate, LENS, out, n_parts=n_parts)
    ref, tol, _, _ = decode_ref(pool, q, gate, LENS, 0, 0, out == BF, out != BF)
    close(got, ref, tol)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("weights", [False, True])
def test_decode_many_sequences(cuda, weights):
    """More sequences than a CTA has threads, long stretches of idle ones in a run; then all idle."""
    g = gen(6)
    B = 1500
    lens = [0 if 300 <= b < 800 or b % 7 == 0 else 1 + b * 37 % 150 for b in range(B)]
    lens[600], lens[-1] = 700, 0
    pool = Pool(g, lens, 2, 16)
    q = normal(g, B, 4, HD)
    w = torch.zeros(B, 2, pool.max_pages * 16, device="cuda") if weights else None
    got = run_decode(pool, q, None, lens, torch.float32, weights=w)
    ref, tol, sums, stol = decode_ref(pool, q, None, lens, 0, 0, False, True)
    close(got, ref, tol)
    assert (got[torch.tensor(lens) == 0] == 0).all()
    if weights:
        close(w, sums, stol)
    got = run_decode(pool, q, None, [0] * B, BF, weights=w)
    assert (got == 0).all()
    if weights:
        close(w, sums, stol)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 4), (128, 130), (129, 1),
                                          (300, 0), (5000, 4)])
@pytest.mark.parametrize("ps,n_parts", [(16, 0), (64, 2), (256, 1)])
def test_decode_window(cuda, window, sinks, ps, n_parts):
    """Pages that no token sees are freed (-1) and what they held is NaN."""
    g = gen(2)
    pool = Pool(g, LENS, 4, ps)
    for b, n in enumerate(LENS):
        s = set(seen(n, window, sinks))
        for j in range(n):
            if j not in s:
                page, row = pool.where(b, [j])
                pool.k[page, :, row] = float("nan")
                pool.v[page, :, row] = float("inf")
        for p in range((n + ps - 1) // ps):
            if not s & set(range(p * ps, p * ps + ps)):
                pool.table[b, p] = -1
    q = normal(g, len(LENS), 24, HD)
    got = run_decode(pool, q, None, LENS, torch.float32, window, sinks, n_parts=n_parts)
    ref, tol, _, _ = decode_ref(pool, q, None, LENS, window, sinks, False, True)
    close(got, ref, tol)


@pytest.mark.parametrize("nq,nkv", [(1, 1), (8, 8), (4, 2), (3, 1), (8, 2), (5, 1), (24, 4), (7, 1),
                                    (16, 2)])
@pytest.mark.parametrize("out,gate", [(torch.float32, BF), (BF, torch.float32), (BF, None)])
def test_decode_heads_and_types(cuda, nq, nkv, out, gate):
    g = gen(3)
    lens = [77, 640, 5]
    pool = Pool(g, lens, nkv, 32)
    q = normal(g, 3, nq, HD)
    gt = None if gate is None else normal(g, 3, nq, HD).to(gate)
    for weights in (None, torch.zeros(3, nkv, pool.max_pages * 32, device="cuda")):
        got = run_decode(pool, q, gt, lens, out, weights=weights)
        ref, tol, sums, stol = decode_ref(pool, q, gt, lens, 0, 0, out == BF,
                                          out != BF or weights is not None)
        close(got, ref, tol)
        if weights is not None:
            close(weights, sums, stol)


@pytest.mark.parametrize("n_parts", [0, 1, 5])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 3)])
def test_decode_weight_sums(cuda, window, sinks, n_parts):
    """The sums grow by each slot's weights, call by call, and stay as they were elsewhere."""
    g = gen(4)
    pool = Pool(g, LENS, 4, 64)
    q = normal(g, len(LENS), 24, HD)
    w = normal(g, len(LENS), 4, pool.max_pages * 64).abs()
    before = w.clone()
    for step in (1, 2):
        run_decode(pool, q, None, LENS, torch.float32, window, sinks, w, n_parts)
        _, _, sums, stol = decode_ref(pool, q, None, LENS, window, sinks, False, True)
        ref = before.double() + step * sums
        close(w, ref, step * stol + 2 * U * ref)
        same = sums == 0
        assert torch.equal(w[same], before[same])


def test_decode_scores_far_apart(cuda):
    """One slot far above all others (weights that underflow), and scores all equal."""
    g = gen(5)
    pool = Pool(g, [400, 400], 1, 16)
    q = normal(g, 2, 6, HD)
    page, row = pool.where(0, [333])
    pool.k[page, :, row] = (q[0, :1] * 8).to(BF)
    page, row = pool.where(1, torch.arange(400))
    pool.k[page, :, row] = 0
    got = run_decode(pool, q, None, [400, 400], torch.float32)
    ref, tol, _, _ = decode_ref(pool, q, None, [400, 400], 0, 0, False, True)
    close(got, ref, tol)


def test_decode_bad_tables_are_reported(cuda):
    """A page or a length outside its table: status 3, the other sequences right."""
    g = gen(6)
    lens = [100, 100, 100]
    pool = Pool(g, lens, 4, 16)
    q = normal(g, 3, 24, HD)
    ref, tol, _, _ = decode_ref(pool, q, None, lens, 0, 0, False, True)
    ws = torch.empty(ops.gqa_paged_workspace_bytes(3, 24, 4, HD, pool.max_pages * 16),
                     dtype=torch.uint8, device="cuda")
    out = torch.empty(3, 24, HD, device="cuda")
    for page, lens_bad in ((-1, lens), (len(pool.k), lens), (2 ** 31 - 1, lens),
                           (None, [100, 10 ** 6, 100]), (None, [100, -5, 100])):
        table = pool.table.clone()
        if page is not None:
            table[1, 2] = page
        ops.gqa_paged_decode(q, None, pool.k, pool.v, table, i32(lens_bad), out, ws)
        assert ops.device_status() == 3
        close(out[[0, 2]], ref[[0, 2]], tol[[0, 2]])


def test_decode_long_cache(cuda):
    """A pool whose rows pass 2^22 and whose byte offsets pass 32 bits, seen at its far end."""
    g = gen(7)
    n, ps = 2_400_000, 256
    pool = Pool(g, [5], 1, ps, max_pages=n // ps + 1)
    k = torch.zeros(n // ps + 1, 1, ps, HD, device="cuda", dtype=BF)
    v = torch.zeros_like(k)
    pool.k, pool.v = k, v
    pool.table = torch.arange(n // ps, -1, -1, dtype=torch.int32, device="cuda").view(1, -1)
    tail = torch.arange(n - 700, n)
    page, row = pool.where(0, tail)
    k[page, :, row], v[page, :, row] = normal(g, 700, 1, HD).to(BF), normal(g, 700, 1, HD).to(BF)
    q = normal(g, 1, 6, HD)
    w = torch.zeros(1, 1, pool.max_pages * ps, device="cuda")
    for window in (0, 650):
        w.zero_()
        got = run_decode(pool, q, None, [n], torch.float32, window=window, weights=w)
        ref, tol, sums, stol = decode_ref(pool, q, None, [n], window, 0, False, True)
        close(got, ref, tol)
        close(w, sums, stol + 1e-30)


# ------------------------------------------------------------------------------ append
def append_ref(x, w, one_p, rope, pos):
    y = x.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6)
    y = y * (w.double() + (1 if one_p else 0))
    t = rope.double()[pos.long()][:, None]
    r = rope.shape[1]
    a, b, c, s = y[..., :r // 2], y[..., r // 2:r], t[..., :r // 2], t[..., r // 2:]
    return torch.cat([a * c - b * s, a * s + b * c, y[..., r:]], -1)


@pytest.mark.parametrize("n", [1, 3, 37])
@pytest.mark.parametrize("act,q_type", [(BF, torch.float32), (torch.float32, BF), (BF, BF)])
@pytest.mark.parametrize("one_p", [False, True])
def test_append_rows(cuda, n, act, q_type, one_p):
    """Rows within rounding of the formula (a few fp32 steps, half a bf16 step when rounded);
    everything else in the pool as it was; idle lanes store nothing."""
    g = gen(8)
    nq, nkv, ps, start = 24, 4, 32, 70
    rope = ops.rope_table(512, 64)
    pool = Pool(g, [start + n, 200], nkv, ps)
    k0, v0 = pool.k.clone(), pool.v.clone()
    q_in, k_in, v_in = (normal(g, n, m, HD).to(act) for m in (nq, nkv, nkv))
    qw, kw = (normal(g, HD) * 0.1 + (0 if one_p else 1) for _ in range(2))
    slots = torch.arange(start, start + n, dtype=torch.int32, device="cuda")
    pos = slots + 100
    if n > 2:
        slots[1] = -1
    q = torch.empty(n, nq, HD, device="cuda", dtype=q_type)
    ops.gqa_paged_append(q_in, k_in, v_in, qw, kw, rope, pos, slots, pool.table, pool.k, pool.v, q,
                         seq=torch.zeros_like(slots), norm_one_plus=one_p)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    # mean of squares, square root, two products and the rotation: 24 fp32 roundings in all,
    # relative to the larger of a rotated pair
    def check(got, x, w, bf):
        ref = append_ref(x, w, one_p, rope, pos)
        size = ref.abs()
        size[..., :64] = (ref[..., :32].square() + ref[..., 32:64].square()).sqrt().repeat(1, 1, 2)
        close(got, ref, 24 * U * size + (H * ref.abs() if bf else 0))
    check(q, q_in, qw, q_type == BF)
    live = slots >= 0
    page, row = pool.where(0, slots[live])
    kk = torch.zeros(n, nkv, HD, device="cuda", dtype=torch.float64)
    kk[live] = pool.k[page, :, row].double()
    ref = append_ref(k_in, kw, one_p, rope, pos)
    kk[~live] = ref[~live]
    check(kk, k_in, kw, True)
    assert torch.equal(pool.v[page, :, row], v_in[live].to(BF))
    k0[page, :, row], v0[page, :, row] = pool.k[page, :, row], pool.v[page, :, row]
    for a, b in ((k0, pool.k), (v0, pool.v)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_append_matches_the_contiguous_append(cuda):
    """The same tokens through gqa_append: the V rows equal bit for bit, q within fp32 rounding
    and K within a bf16 step (the two sum the squares in different orders)."""
    g = gen(9)
    B, nq, nkv, ps, cap = 3, 24, 4, 16, 64
    rope = ops.rope_table(512, 64)
    q_in, k_in, v_in = (normal(g, B, m, HD).to(BF) for m in (nq, nkv, nkv))
    w = 1 + 0.02 * normal(g, HD)
    pos = i32([0, 17, 63])
    kc, vc = (torch.zeros(B, nkv, cap, HD, device="cuda", dtype=BF) for _ in range(2))
    q0, q1 = (torch.empty(B, nq, HD, device="cuda") for _ in range(2))
    ops.gqa_append(q_in, k_in, v_in, w, w, rope, pos, kc, vc, q0)
    pool = Pool(g, [64] * B, nkv, ps)
    ops.gqa_paged_append(q_in, k_in, v_in, w, w, rope, pos, pos, pool.table, pool.k, pool.v, q1)
    close(q1, q0.double(), 48 * U * q0.double().abs().amax(-1, keepdim=True))
    for b, p in enumerate(pos.tolist()):
        k, v = pool.rows(b, [p])
        assert torch.equal(v[:, 0], vc[b, :, p].double())
        close(k[:, 0], kc[b, :, p].double(), 2 * H * kc[b, :, p].double().abs() + 1e-30)


def test_append_reports_what_it_cannot_store(cuda):
    g = gen(10)
    n, nq, nkv, ps = 6, 6, 1, 16
    pool = Pool(g, [64, 64], nkv, ps)
    pool.table[1, 1] = len(pool.k)
    k0 = pool.k.clone()
    rope = ops.rope_table(32, 64)
    q_in, k_in = normal(g, n, nq, HD), normal(g, n, nkv, HD)
    w, q = torch.ones(HD, device="cuda"), torch.empty(n, nq, HD, device="cuda")
    # sequence below 0, behind the last; slot behind the table; a page that is none
    ops.gqa_paged_append(q_in, k_in, k_in, w, w, rope, i32([0] * n), i32([1, 1, 64, 16, 5, -7]),
                         pool.table, pool.k, pool.v, q, seq=i32([-1, 2, 0, 1, 0, 0]))
    assert ops.device_status() == 3
    page, row = pool.where(0, [5])
    k0[page, :, row] = pool.k[page, :, row]
    assert torch.equal(k0.view(torch.int16), pool.k.view(torch.int16))
    ops.gqa_paged_append(q_in, k_in, k_in, w, w, rope, i32([0, 1, 2, 3, 31, 32]), i32([-1] * n),
                         pool.table, pool.k, pool.v, q, seq=i32([0] * n))
    assert ops.device_status() == 3  # a position behind the rope table


# ------------------------------------------------------------------------------ prompt
def prompt_ref(pool, q, gate, s0, window, sinks):
    T, nq, nkv = q.shape[0], q.shape[1], pool.nkv
    G = nq // nkv
    n = s0 + T
    at = torch.arange(s0, n, device="cuda")
    j = torch.arange(n, device="cuda")
    mask = j <= at[:, None]
    if window:
        mask &= (j > at[:, None] - window) | (j < sinks)
    used = mask.any(0).nonzero().flatten()
    k, v = pool.rows(0, used)
    qq = q.view(T, nkv, G, HD).permute(1, 2, 0, 3).reshape(nkv, G * T, HD)
    o, _, av, A = attend(qq, k, v, mask[:, used].repeat(G, 1))
    dp = 2 * 256 * U * A + 16 * U
    tol = (2 * dp + H + 256 * U) * av
    back = lambda x: x.view(nkv, G, T, HD).permute(2, 0, 1, 3).reshape(T, nq, HD)  # noqa: E731
    o, tol = back(o), back(tol)
    if gate is not None:
        s = torch.sigmoid(gate.double())
        o, tol = o * s, tol * s + 2.0 ** -20 * (o * s).abs()
    return o, tol * (1 + H) + H * o.abs() + 1e-30


def run_prompt(pool, q, gate, s0, window=0, sinks=0, stream=None):
    ws = torch.empty(ops.gqa_paged_prefill_workspace_bytes(pool.nkv, HD), dtype=torch.uint8,
                     device="cuda")
    out = torch.full(q.shape, float("nan"), device="cuda", dtype=BF)
    ops.gqa_paged_prefill(q, gate, pool.k, pool.v, pool.table[0], out, ws, s0=s0, window=window,
                          sinks=sinks, stream=stream)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    return out


@pytest.mark.parametrize("T,s0", [(1, 0), (1, 200), (2, 127), (63, 1), (64, 64), (128, 0), (129, 0),
                                  (130, 126), (300, 1000), (513, 63)])
@pytest.mark.parametrize("ps", [16, 64, 256])
def test_prompt_causal(cuda, T, s0, ps):
    g = gen(11)
    pool = Pool(g, [s0 + T], 4, ps)
    q, gate = normal(g, T, 24, HD).to(BF), normal(g, T, 24, HD).to(BF)
    k0 = pool.k.clone()
    got = run_prompt(pool, q, gate, s0)
    close(got, *prompt_ref(pool, q, gate, s0, 0, 0))
    assert torch.equal(k0.view(torch.int16), pool.k.view(torch.int16))


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 4), (128, 0), (129, 130), (250, 4),
                                          (600, 64), (9999, 4)])
@pytest.mark.parametrize("T,s0,ps", [(1, 999, 16), (500, 0, 32), (300, 700, 128), (257, 333, 16)])
def test_prompt_window(cuda, window, sinks, T, s0, ps):
    """Pages that no token of the call sees are freed."""
    g = gen(12)
    n = s0 + T
    pool = Pool(g, [n], 2, ps)
    lo = max(s0 + 1 - window, 0)
    for p in range((n + ps - 1) // ps):
        if p * ps + ps <= lo and p * ps >= sinks:
            pool.k[pool.table[0, p].long()] = float("nan")
            pool.v[pool.table[0, p].long()] = float("nan")
            pool.table[0, p] = -1
    q = normal(g, T, 12, HD).to(BF)
    got = run_prompt(pool, q, None, s0, window, sinks)
    close(got, *prompt_ref(pool, q, None, s0, window, sinks))


@pytest.mark.parametrize("nq,nkv", [(1, 1), (2, 2), (6, 2), (5, 1), (7, 1), (8, 1), (24, 4)])
def test_prompt_heads(cuda, nq, nkv):
    g = gen(13)
    pool = Pool(g, [290], nkv, 32)
    q, gate = normal(g, 200, nq, HD).to(BF), normal(g, 200, nq, HD).to(BF)
    for window, sinks in ((0, 0), (40, 2)):
        got = run_prompt(pool, q, gate, 90, window, sinks)
        close(got, *prompt_ref(pool, q, gate, 90, window, sinks))


@pytest.mark.parametrize("nq,nkv", [(24, 4), (5, 1), (2, 2)])
@pytest.mark.parametrize("T,s0,window,sinks", [(1, 20000, 0, 0), (65, 7001, 0, 0), (300, 9000, 0, 0),
                                               (200, 12000, 5000, 300), (1, 9000, 8999, 1),
                                               (1500, 3000, 0, 0), (3000, 0, 2500, 4)])
def test_prompt_few_rows_over_many_slots(cuda, nq, nkv, T, s0, window, sinks):
    """Key tiles of a pair spread over several clusters, whose parts are joined; with a window
    some rows see nothing of a part."""
    g = gen(23)
    pool = Pool(g, [s0 + T], nkv, 64)
    q, gate = normal(g, T, nq, HD).to(BF), normal(g, T, nq, HD).to(BF)
    for gt in (gate, None):
        got = run_prompt(pool, q, gt, s0, window, sinks)
        close(got, *prompt_ref(pool, q, gt, s0, window, sinks))


def test_prompts_replay_and_overlap(cuda):
    """Two captured prompts (one of them joined from parts), replayed at once on streams and
    workspaces of their own with other rows in the same buffers; a table row that is not the first."""
    g = gen(24)
    cases = []
    for T, s0, b in ((200, 100, 0), (3, 5000, 1)):
        pool = Pool(g, [40, s0 + T] if b else [s0 + T, 40], 4, 64)
        q, gate = normal(g, T, 24, HD).to(BF), normal(g, T, 24, HD).to(BF)
        out = torch.empty_like(q)
        ws = torch.empty(ops.gqa_paged_prefill_workspace_bytes(4, HD), dtype=torch.uint8, device="cuda")

        def call(pool=pool, q=q, gate=gate, out=out, ws=ws, s0=s0, b=b):
            ops.gqa_paged_prefill(q, gate, pool.k, pool.v, pool.table[b], out, ws, s0=s0)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        cases.append((pool, q, gate, out, s0, b, ws, graph, torch.cuda.Stream()))
    for pool, q, gate, out, *_ in cases:
        q.copy_(normal(g, *q.shape))
        out.fill_(float("nan"))
    torch.cuda.synchronize()
    for _ in range(10):
        for *_, graph, stream in cases:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    for pool, q, gate, out, s0, b, *_ in cases:
        pool.table = pool.table[b:].clone()  # of prompt_ref's sequence 0
        close(out, *prompt_ref(pool, q, gate, s0, 0, 0))


def test_prompt_bad_page_is_reported(cuda):
    g = gen(14)
    pool = Pool(g, [300], 4, 16)
    q = normal(g, 100, 24, HD).to(BF)
    ws = torch.empty(ops.gqa_paged_prefill_workspace_bytes(4, HD), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    for page in (-1, len(pool.k), 2 ** 31 - 1):
        for at in (2, 18):
            table = pool.table[0].clone()
            table[at] = page
            ops.gqa_paged_prefill(q, None, pool.k, pool.v, table, out, ws, s0=200)
            assert ops.device_status() == 3


# ------------------------------------------------------------------------------- evict
def evict_ref(sums, n, keep, sinks, recent):
    """Kept slots of one (sequence, head), by sorting."""
    if n <= keep:
        return list(range(n))
    s = np.where(np.isnan(sums), -np.inf, sums)
    mid = sorted(range(sinks, n - recent), key=lambda j: (-s[j], j))[:keep - sinks - recent]
    return [*range(sinks), *sorted(mid), *range(n - recent, n)]


@pytest.mark.parametrize("ps", [16, 64])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 1, 0), (20, 4, 16), (33, 4, 8),
                                               (128, 0, 0), (300, 16, 100), (1100, 4, 5)])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict(cuda, ps, keep, sinks, recent, kind):
    g = gen(15)
    lens = [0, 1, 19, 33, 34, 129, 300, 1000, 1099]
    B, nkv = len(lens), 2
    pool = Pool(g, lens, nkv, ps, spare=B * ((keep + ps - 1) // ps + 1) + 2)
    S = pool.max_pages * ps
    sums = torch.rand(B, nkv, S, generator=g, device="cuda")
    if kind == "ties":
        sums = (sums * 4).floor()
    if kind == "odd":  # infinities, NaN, zeros of both signs, subnormals
        pick = torch.randint(0, 6, sums.shape, generator=g, device="cuda")
        for i, x in enumerate((float("inf"), float("nan"), -0.0, 0.0, 1e-42)):
            sums[pick == i] = x
    mo = (keep + ps - 1) // ps + 1
    dst = pool.spare[:B * mo].view(B, mo).contiguous()
    k0, v0 = pool.k.clone(), pool.v.clone()
    lens_out, kept = i32([-9] * B), torch.full((B, nkv, keep), -9, dtype=torch.int32, device="cuda")
    sums_out = torch.full((B, nkv, mo * ps), float("nan"), device="cuda")
    ops.kv_evict(pool.k, pool.v, pool.table, i32(lens), sums, dst, lens_out, sums_out, kept, keep,
                 sinks=sinks, recent=recent)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    assert lens_out.tolist() == [min(n, keep) for n in lens]
    want_sums = torch.zeros_like(sums_out)
    for b, n in enumerate(lens):
        for h in range(nkv):
            ref = evict_ref(sums[b, h].cpu().numpy(), n, keep, sinks, recent)
            assert kept[b, h].tolist() == ref + [-1] * (keep - len(ref))
            at = torch.tensor(ref, dtype=torch.long, device="cuda")
            j = torch.arange(len(ref), device="cuda")
            want_sums[b, h, :len(ref)] = sums[b, h, at]
            page, row = pool.where(b, at)
            to = dst[b].long()[j // ps]
            for p, p0 in ((pool.k, k0), (pool.v, v0)):
                assert torch.equal(p[to, h, j % ps], p0[page, h, row])
                p0[to, h, j % ps] = p0[page, h, row]
    assert torch.equal(want_sums.view(torch.int32), sums_out.view(torch.int32))
    for p, p0 in ((pool.k, k0), (pool.v, v0)):  # nothing else was written
        assert torch.equal(p.view(torch.int16), p0.view(torch.int16))


@pytest.mark.parametrize("n", [70_001, 262_144])
def test_evict_long(cuda, n):
    g = gen(16)
    ps, keep = 256, 5000
    pool = Pool(g, [n], 1, ps, spare=(keep + ps - 1) // ps)
    sums = torch.rand(1, 1, pool.max_pages * ps, generator=g, device="cuda") ** 4
    dst = pool.spare.view(1, -1).contiguous()
    lens_out, kept = i32([0]), torch.zeros(1, 1, keep, dtype=torch.int32, device="cuda")
    sums_out = torch.empty(1, 1, dst.shape[1] * ps, device="cuda")
    ops.kv_evict(pool.k, pool.v, pool.table, i32([n]), sums, dst, lens_out, sums_out, kept, keep,
                 sinks=4, recent=64)
    assert kept[0, 0].tolist() == evict_ref(sums[0, 0].cpu().numpy(), n, keep, 4, 64)
    page, row = pool.where(0, kept[0, 0])
    j = torch.arange(keep, device="cuda")
    assert torch.equal(pool.k[dst[0].long()[j // ps], 0, j % ps], pool.k[page, 0, row])
    assert ops.device_status() == 0


def test_evict_bad_pages_are_reported(cuda):
    g = gen(17)
    pool = Pool(g, [100, 100], 1, 16, spare=8)
    sums = torch.rand(2, 1, pool.max_pages * 16, generator=g, device="cuda")
    dst = pool.spare[:4].view(2, 2).contiguous()
    lens_out, kept = i32([0, 0]), torch.zeros(2, 1, 32, dtype=torch.int32, device="cuda")
    sums_out = torch.empty(2, 1, 32, device="cuda")
    for table, out in ((-1, None), (len(pool.k), None), (None, -3), (None, len(pool.k))):
        t, d = pool.table.clone(), dst.clone()
        if table is not None:
            t[0] = table
        if out is not None:
            d[0, 1] = out
        before = pool.k.clone()
        ops.kv_evict(pool.k, pool.v, t, i32([100, 100]), sums, d, lens_out, sums_out, kept, 32)
        assert ops.device_status() == 3
        own = torch.zeros(len(pool.k), dtype=torch.bool, device="cuda")
        own[dst.flatten().long()] = True
        assert torch.equal(before.view(torch.int16)[~own], pool.k.view(torch.int16)[~own])


# ---------------------------------------------------------------------------- together
def test_prompt_decode_evict_decode(cuda):
    """A run as they are used: a prompt enters and is attended to, tokens are decoded with
    their weights summed, the cache is cut back, and decoding goes on over what is left; every
    step against the formulas over the rows that the pool then holds."""
    g = gen(18)
    nq, nkv, ps, T, steps, keep = 24, 4, 32, 150, 40, 96
    rope = ops.rope_table(512, 64)
    w = 1 + 0.02 * normal(g, HD)
    pool = Pool(g, [T + steps], nkv, ps, spare=8)
    pool.k.fill_(float("nan"))
    pool.v.fill_(float("nan"))
    toks = [normal(g, T + steps + 20, m, HD).to(BF) for m in (nq, nkv, nkv, nq)]
    slots = torch.arange(T, dtype=torch.int32, device="cuda")
    q = torch.empty(T, nq, HD, device="cuda", dtype=BF)
    ops.gqa_paged_append(*(t[:T] for t in toks[:3]), w, w, rope, slots, slots, pool.table, pool.k,
                         pool.v, q, seq=torch.zeros_like(slots))
    got = run_prompt(pool, q, toks[3][:T], 0)
    close(got, *prompt_ref(pool, q, toks[3][:T], 0, 0, 0))
    sums = torch.zeros(1, nkv, pool.max_pages * ps, device="cuda")
    model = torch.zeros_like(sums, dtype=torch.float64)
    qd = torch.empty(1, nq, HD, device="cuda")

    def step(t, n):
        """Token t enters as the n-th slot."""
        ops.gqa_paged_append(*(x[t:t + 1] for x in toks[:3]), w, w, rope, i32([t]), i32([n - 1]),
                             pool.table, pool.k, pool.v, qd)
        out = run_decode(pool, qd, toks[3][t:t + 1], [n], BF, weights=sums)
        ref, tol, add, stol = decode_ref(pool, qd, toks[3][t:t + 1], [n], 0, 0, True, True)
        close(out, ref, tol)
        model.add_(add)
        # each addition rounds once more
        close(sums, model, (t + 1) * (stol.max() + U * model))
    for i in range(steps):
        step(T + i, T + i + 1)
    mo = 4
    dst = pool.spare[:mo].view(1, mo).contiguous()
    lens_out, kept = i32([0]), torch.zeros(1, nkv, keep, dtype=torch.int32, device="cuda")
    sums_out = torch.empty(1, nkv, mo * ps, device="cuda")
    ops.kv_evict(pool.k, pool.v, pool.table, i32([T + steps]), sums, dst, lens_out, sums_out, kept,
                 keep, sinks=4, recent=16)
    assert lens_out.tolist() == [keep]
    for h in range(nkv):
        assert kept[0, h].tolist() == evict_ref(sums[0, h].cpu().numpy(), T + steps, keep, 4, 16)
    pool.table, pool.max_pages, sums, model = dst, mo, sums_out, sums_out.double()
    for i in range(20):
        step(T + steps + i, keep + i + 1)


def test_steps_replay_from_a_graph(cuda):
    """Append, decode with weights and evict captured into two graphs on workspaces of their own,
    replayed: the results of the calls made one by one."""
    g = gen(19)
    B, nq, nkv, ps = 3, 24, 4, 64
    lens = [260, 100, 1]
    rope = ops.rope_table(512, 64)
    w = 1 + 0.02 * normal(g, HD)
    x = [normal(g, B, m, HD).to(BF) for m in (nq, nkv, nkv, nq)]

    def make():
        st = gen(20)
        pool = Pool(st, [n + 8 for n in lens], nkv, ps, spare=B * 2)
        s = dict(pool=pool, lens=i32(lens), pos=i32([n - 1 for n in lens]),
                 q=torch.empty(B, nq, HD, device="cuda"),
                 out=torch.empty(B, nq, HD, device="cuda", dtype=BF),
                 sums=torch.zeros(B, nkv, pool.max_pages * ps, device="cuda"),
                 lens2=i32([0] * B), kept=torch.zeros(B, nkv, 90, dtype=torch.int32, device="cuda"),
                 sums2=torch.empty(B, nkv, 2 * ps, device="cuda"),
                 dst=pool.spare[:2 * B].view(B, 2).contiguous())
        s["ws"] = torch.empty(ops.gqa_paged_workspace_bytes(B, nq, nkv, HD, pool.max_pages * ps,
                                                            weights=True),
                              dtype=torch.uint8, device="cuda")
        return s

    def step(s):
        p = s["pool"]
        ops.gqa_paged_append(*x[:3], w, w, rope, s["pos"], s["pos"], p.table, p.k, p.v, s["q"])
        ops.gqa_paged_decode(s["q"], x[3], p.k, p.v, p.table, s["lens"], s["out"], s["ws"],
                             weight_sum=s["sums"])
        ops.kv_evict(p.k, p.v, p.table, s["lens"], s["sums"], s["dst"], s["lens2"], s["sums2"],
                     s["kept"], 90, sinks=2, recent=10)
        ops.add_int(s["pos"], 1)
        ops.add_int(s["lens"], 1)
    eager, graphed = make(), [make(), make()]
    step(make())  # module loading, outside the capture
    torch.cuda.synchronize()
    graphs = []
    for s in graphed:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step(s)
        graphs.append(gr)
    for _ in range(4):
        step(eager)
        for gr in graphs:
            gr.replay()
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    for s in graphed:
        for key in ("out", "sums", "lens2", "kept", "sums2", "lens"):
            assert torch.equal(s[key], eager[key]), key


def test_on_another_stream(cuda):
    """The calls run on the stream they are given, behind what it already holds."""
    g = gen(21)
    pool = Pool(g, [500], 4, 16)
    q = normal(g, 1, 24, HD)
    ref, tol, _, _ = decode_ref(pool, q, None, [500], 0, 0, False, True)
    side = torch.cuda.Stream()
    late = torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late.copy_(q)
    got = run_decode(pool, late, None, [500], torch.float32, stream=side)
    close(got, ref, tol)


def test_two_calls_at_once(cuda):
    """Two decodes that overlap on the GPU, each on a stream and a workspace of its own."""
    g = gen(22)
    pools = [Pool(g, [700, 90], 4, 32), Pool(g, [333, 1], 4, 64)]
    lens = [[700, 90], [333, 1]]
    qs = [normal(g, 2, 24, HD) for _ in pools]
    ws = [torch.empty(ops.gqa_paged_workspace_bytes(2, 24, 4, HD, p.max_pages * p.ps),
                      dtype=torch.uint8, device="cuda") for p in pools]
    outs = [torch.empty(2, 24, HD, device="cuda") for _ in pools]
    lt = [i32(x) for x in lens]
    streams = [torch.cuda.Stream() for _ in pools]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, q, w, o, n, s in zip(pools, qs, ws, outs, lt, streams):
            ops.gqa_paged_decode(q, None, p.k, p.v, p.table, n, o, w, stream=s)
    torch.cuda.synchronize()
    for p, q, o, n in zip(pools, qs, outs, lens):
        ref, tol, _, _ = decode_ref(p, q, None, n, 0, 0, False, True)
        close(o, ref, tol)
    assert ops.device_status() == 0


# ------------------------------------------------------------------ the layer over the cache
def gqa_layer(seed, H=512, nq=12, nkv=2):
    """A GQA layer with fp32 weights, as uploaded rows."""
    from vx27_b200.layer import GQALayer, PackedLinear
    g = gen(seed)

    def lin(rows, cols):
        w = normal(g, rows, cols) / cols ** 0.5
        return PackedLinear(w.view(torch.uint8), ops.PMAT_F32, rows, cols)
    return GQALayer(lin(nq * 2 * HD, H), lin(nkv * HD, H), lin(nkv * HD, H), lin(H, nq * HD),
                    0.02 * normal(g, HD), 0.02 * normal(g, HD), ops.rope_table(512), nq, nkv)


def test_layer_over_pages_matches_the_contiguous_cache(cuda):
    """GQALayer.step_paged against GQALayer.step, token by token, an idle lane among them: the
    same projections, so the outputs differ by the attention's and norms' rounding (both within
    1e-5 of the formulas; 1e-4 of the largest value leaves room for the K rows that round to
    the other bf16 neighbour, one in ~1000 by 2^-8 of its size)."""
    from vx27_b200.paged import PagedKV
    layer, B, cap, H = gqa_layer(30), 3, 64, 512
    g = gen(31)
    kc, vc = (torch.zeros(2, 2, cap, HD, device="cuda", dtype=BF) for _ in range(2))
    ws = torch.empty(ops.gqa_workspace_bytes(2, 12, 2, HD, cap) // 4 + 1, device="cuda")
    cache = PagedKV(1, B, 12, 4, 16, 2)
    cw = cache.workspace(12)
    for t in range(40):
        x = normal(g, B, H)
        at = cache.extend({0: 1, 2: 1})
        assert at[0] == at[2] == (t, t)
        got = layer.step_paged(x, cache, 0, cw)
        ref = layer.step(x[[0, 2]], kc, vc, i32([t, t]), ws)
        assert float((got[[0, 2]] - ref).abs().max()) <= 1e-4 * float(ref.abs().max())
        assert (got[1] == 0).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("window,sinks,weights", [(0, 0, True), (50, 4, False)])
def test_layer_prompt_then_steps(cuda, window, sinks, weights):
    """A prompt through prompt_paged, in two parts, then tokens through step_paged, with pages
    freed behind a window or the cache cut back by evict, against the layer's formulas in 64
    bits over the rows that the cache then holds (bf16 results in prompts: 2^-7 of the largest
    value; 1e-4 in steps, as above)."""
    from vx27_b200.paged import PagedKV
    layer, H, T, nkv, nq = gqa_layer(32), 512, 150, 2, 12
    g = gen(33)
    cache = PagedKV(1, 2, 40, 20, 16, nkv, window=window, sinks=sinks, weights=weights)
    ws = cache.workspace(nq)
    wd = [m.W.view(torch.float32).view(m.rows, m.cols).double() for m in (layer.q, layer.o)]

    def want(x, n0):
        """x [n, H] at slots n0 ..: the formulas, the cache's own K and V rows."""
        qg = (x.double() @ wd[0].T).view(len(x), nq, 2, HD)
        q = append_ref(qg[:, :, 0], layer.q_norm_w, True, layer.rope, torch.tensor(at_pos))
        out = []
        for i in range(len(x)):
            page = cache.table[seq].long()
            s = torch.tensor(seen(n0 + i + 1, window, sinks), device="cuda")
            k = cache.k[0][page[s // 16], :, s % 16].double().transpose(0, 1)
            v = cache.v[0][page[s // 16], :, s % 16].double().transpose(0, 1)
            o = attend(q[i].view(nkv, -1, HD), k, v)[0].reshape(nq, HD)
            out.append((o * torch.sigmoid(qg[i, :, 1])).flatten() @ wd[1].T)
        return torch.stack(out)
    seq, done = 1, 0
    for n in (T - 33, 33):
        x = normal(g, n, H)
        slot, pos = cache.extend({seq: n})[seq]
        assert (slot, pos) == (done, done)
        got = layer.prompt_paged(x, cache, 0, seq, slot, pos, ws)
        at_pos = list(range(pos, pos + n))
        ref = want(x, slot)
        assert float((got - ref).abs().max()) <= 2.0 ** -7 * float(ref.abs().max())
        done += n
    free = cache.free_pages
    for t in range(40):
        if weights and t == 20:
            cut, kept = cache.evict(64, sinks=4, recent=16)
            assert cut == [seq] and kept.shape == (1, 1, nkv, 64) and cache.length(seq) == 64
            assert cache.free_pages == 36 and cache.position(seq) == T + 20
        x = normal(g, 2, H)
        slot, pos = cache.extend({seq: 1})[seq]
        got = layer.step_paged(x, cache, 0, ws)
        at_pos = [pos]
        ref = want(x[1:], slot)
        assert float((got[1] - ref[0]).abs().max()) <= 1e-4 * float(ref.abs().max())
        assert (got[0] == 0).all()
    if window:
        assert cache.free_pages > free  # the prompt's pages behind the window
    if weights:  # each token hands out 1 per head, 6 heads a KV head; eviction drops some
        total = cache.sums[0, seq].sum(-1)
        assert ((total > 6 * 20 - 0.01) & (total < 6 * 40)).all()
    cache.release(seq)
    assert cache.free_pages == 40
    assert ops.device_status() == 0


def test_layer_step_replays_and_leaves_idle_lanes(cuda):
    """A captured step_paged replayed after each extend gives the eager results bit for bit; a
    sequence that an extend leaves out keeps its rows and sums."""
    from vx27_b200.paged import PagedKV
    layer, B, H = gqa_layer(34), 3, 512
    g = gen(35)
    caches = [PagedKV(1, B, 12, 4, 16, 2, weights=True) for _ in range(2)]
    ws = [c.workspace(12) for c in caches]
    prompt, x = normal(g, 30, H), torch.empty(B, H, device="cuda")
    for c, w in zip(caches, ws):
        c.k.zero_()
        c.v.zero_()
        layer.prompt_paged(prompt, c, 0, 1, *c.extend({1: 30})[1], w)
    layer.step_paged(x.zero_(), caches[1], 0, ws[1])  # all lanes idle
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.step_paged(x, caches[1], 0, ws[1])
    for t in range(20):
        tokens = {0: 1} if t % 3 == 0 else {1: 1} if t % 3 == 1 else {0: 1, 1: 1, 2: 1}
        x.copy_(normal(g, B, H))
        rows = {s: caches[1].sums[0, s].clone() for s in range(B) if s not in tokens}
        for c in caches:
            c.extend(tokens)
        ref = layer.step_paged(x, caches[0], 0, ws[0])
        graph.replay()
        assert torch.equal(out, ref)
        for s, before in rows.items():
            assert (out[s] == 0).all() and torch.equal(caches[1].sums[0, s], before)
    for name in ("k", "v", "sums", "table", "lens", "pos", "step"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name
    assert ops.device_status() == 0
