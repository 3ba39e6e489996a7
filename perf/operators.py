"""The operators over the paged key-value cache: their cases, plain forms and 64-bit values.

A cache is a pool of pages, ``k_pages`` and ``v_pages`` bf16 [n_pages][nkv][page_size][256], and
a table ``page_table`` int32 [B][max_pages]: slot s of sequence b is row s % page_size of page
page_table[b][s // page_size]. Four operators use it:

* append   RMSNorm of q and k, rotation of their first 64 dims, k and v into their slots
* decode   attention of one token a sequence over its slots, all of them or the first few
           (sinks) and a window of the last ones; on request the attention each slot got is
           added to a running sum
* prompt   causal attention of T tokens of one sequence over its slots, with the same window
* evict    the slots with the largest sums stay (with the first and the last ones), copied in
           order to other pages

The plain forms compute in 32 bits with elementary torch operations and round once at the end.
"""
import math

import torch

own = False

HD, ROT = 256, 64
EPS = 1e-6


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one sequence takes a token: the smallest call of a decode loop, latency alone
        dict(name="append_one", op="append", n=1, one_seq=False, nq=24, nkv=4, ps=16, first=776,
             act="bf16", q="f32", plus=True),
        # a prompt of 4096 tokens enters the cache behind 1000 earlier slots
        dict(name="append_prompt_4096", op="append", n=4096, one_seq=True, nq=24, nkv=4, ps=64,
             first=1000, act="bf16", q="bf16", plus=True),
        # batch 1 on a short context, pages of 16 that end inside every tile
        dict(name="decode_one_777", op="decode", B=1, L=777, nq=24, nkv=4, ps=16, window=0,
             sinks=0, ragged=False, gate="bf16", out="bf16", weights=False),
        # batch 1 at 8192 positions in fp32, as a whole fp32 layer calls it
        dict(name="decode_one_8192", op="decode", B=1, L=8192, nq=24, nkv=4, ps=64, window=0,
             sinks=0, ragged=False, gate="f32", out="f32", weights=False),
        # a serving batch at mixed lengths up to 4163, idle lanes among them
        dict(name="decode_ragged_128", op="decode", B=128, L=4163, nq=24, nkv=4, ps=64, window=0,
             sinks=0, ragged=True, gate="bf16", out="bf16", weights=False),
        # long sequences whose pages between the sinks and the window are freed
        dict(name="decode_window_256", op="decode", B=256, L=32768, nq=24, nkv=4, ps=32,
             window=1024, sinks=4, ragged=True, gate="bf16", out="bf16", weights=False),
        # a batch that sums its weights for a later eviction
        dict(name="decode_weights_32", op="decode", B=32, L=4163, nq=24, nkv=4, ps=128, window=0,
             sinks=0, ragged=True, gate="f32", out="f32", weights=True),
        # a short odd prompt that continues a cache, pages of 16
        dict(name="prompt_300", op="prompt", T=300, s0=130, nq=24, nkv=4, ps=16, window=0,
             sinks=0, gate=True),
        # a chunk of a long prompt, plain causal
        dict(name="prompt_2048_at_14001", op="prompt", T=2048, s0=14001, nq=24, nkv=4, ps=64,
             window=0, sinks=0, gate=True),
        # a whole long prompt under a window with sinks
        dict(name="prompt_32768_window", op="prompt", T=32768, s0=0, nq=24, nkv=4, ps=128,
             window=4096, sinks=4, gate=True),
        # one sequence cut back to its budget
        dict(name="evict_one", op="evict", B=1, L=5001, keep=2048, sinks=4, recent=256, nkv=4,
             ps=16, ragged=False),
        # a whole batch cut back, the short sequences of it kept whole
        dict(name="evict_64", op="evict", B=64, L=4163, keep=1024, sinks=4, recent=128, nkv=4,
             ps=64, ragged=True),
    ]


HEADS = [(24, 4), (24, 4), (16, 2), (8, 8), (12, 4), (28, 4), (5, 1), (20, 4)]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "decode", "prompt", "prompt", "evict"])
    nq, nkv = rng.choice(HEADS)
    ps = rng.choice([16, 32, 64, 128, 256])
    c = dict(op=op, nq=nq, nkv=nkv, ps=ps)
    if op == "append":
        one_seq = rng.random() < 0.5
        c |= dict(n=_log(rng, 1, 4096 if one_seq else 256), one_seq=one_seq,
                  first=_log(rng, 1, 30000) - 1, act=rng.choice(["bf16", "f32"]),
                  q=rng.choice(["bf16", "f32"]), plus=rng.random() < 0.5)
    elif op == "decode":
        window = rng.choice([0, 0, _log(rng, 1, 4096)])
        B = _log(rng, 1, 256)
        # at most the slots of the largest listed decode, by key-value heads
        slots = 1_000_000 // (B * nkv)
        L = _log(rng, 1, 40000) if window and window <= slots else _log(rng, 1, min(40000, slots))
        c |= dict(B=B, L=L, window=window, sinks=rng.choice([0, 1, 4, 64]) if window else 0,
                  ragged=rng.random() < 0.7, gate=rng.choice(["bf16", "f32", "none"]),
                  out=rng.choice(["bf16", "f32"]), weights=rng.random() < 0.3)
    elif op == "prompt":
        T = _log(rng, 1, 8192)
        window = rng.choice([0, _log(rng, 1, 4096)])
        c |= dict(T=T, s0=rng.choice([0, _log(rng, 1, 8192)]), window=window,
                  sinks=rng.choice([0, 1, 4, 64]) if window else 0, gate=rng.random() < 0.7)
    else:
        del c["nq"]
        B = _log(rng, 1, 64)
        L = _log(rng, 16, min(30000, 1_000_000 // (B * nkv)))
        keep = max(1, int(L * rng.uniform(0.1, 1.1)))
        c |= dict(B=B, L=L, keep=keep, sinks=min(rng.choice([0, 4, 16]), keep // 2),
                  recent=rng.randint(0, keep // 2), ragged=rng.random() < 0.7)
    return c


def _lens(case):
    """Slots that each sequence holds: L for all, or spread over [0, L] with an idle lane (0), a
    single slot and L itself among them."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L] * B
    lens = [1 + (b * 2654435761 + 12345) % (1 << 32) * L // (1 << 32) for b in range(B)]
    lens[0] = L
    if B >= 4:
        lens[1], lens[2] = 0, 1
    return lens


def _seen(n, window, sinks):
    """Slots that a token with n slots behind it (itself included) attends to."""
    return n if not window else min(n, window) + min(sinks, max(n - window, 0))


# ------------------------------------------------------------------------------- work
def work(case):
    size = {"bf16": 2, "f32": 4, "none": 0}
    op, nkv = case["op"], case["nkv"]
    row = HD * 2
    if op == "append":
        n, nq, a = case["n"], case["nq"], size[case["act"]]
        byt = n * HD * ((nq + 2 * nkv) * a + nq * size[case["q"]] + 2 * nkv * 2) + n * (8 + ROT * 4)
        return {"bytes": byt + 2 * HD * 4, "flops": n * (nq + nkv) * (4 * HD + 3 * ROT)}
    if op == "decode":
        nq = case["nq"]
        seen = sum(_seen(n, case["window"], case["sinks"]) for n in _lens(case))
        byt = seen * nkv * 2 * row + case["B"] * nq * HD * (4 + size[case["gate"]] + size[case["out"]])
        if case["weights"]:
            byt += seen * nkv * 8
        return {"bytes": byt + 4 * (case["B"] + seen // case["ps"]), "flops": 4 * seen * nq * HD}
    if op == "prompt":
        T, s0, nq, w, k = case["T"], case["s0"], case["nq"], case["window"], case["sinks"]
        seen = sum(_seen(s0 + t + 1, w, k) for t in range(T))
        held = s0 + T if not w else min(s0 + T, T + w - 1 + k)
        byt = T * nq * HD * 2 * (3 if case["gate"] else 2) + held * nkv * 2 * row
        return {"bytes": byt, "flops": 4 * seen * nq * HD}
    lens = _lens(case)
    kept = sum(min(n, case["keep"]) for n in lens)
    byt = nkv * (kept * (2 * 2 * row + 8 + 4) + sum(lens) * 4)
    return {"bytes": byt, "flops": nkv * sum(lens)}


# ----------------------------------------------------------------------------- inputs
def _dt(name):
    return {"bf16": torch.bfloat16, "f32": torch.float32}[name]


def _pool(n_pages, case, g):
    shape = (max(n_pages, 1), case["nkv"], case["ps"], HD)
    return [torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]


def _table(live, g):
    """A page of its own, in random order, for every entry of live (bool [B][max_pages]); -1
    elsewhere."""
    table = torch.full(live.shape, -1, dtype=torch.int32, device="cuda")
    n = int(live.sum())
    table[live] = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    return table, n


def _live(lens, ps, window, sinks):
    """Which pages hold a slot that is attended to."""
    n = max((max(lens) + ps - 1) // ps, 1)
    first = torch.arange(n, device="cuda") * ps
    lens = torch.tensor(lens, device="cuda")[:, None]
    live = first < lens
    if window:
        live &= (first + ps > lens - window) | (first < sinks)
    return live


def _rope(n):
    """[n][64]: cosines then sines of pos * 1e7^(-i/32)."""
    f = 1e7 ** (-torch.arange(ROT // 2, device="cuda", dtype=torch.float64) / (ROT // 2))
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    st = dict(case=case)
    op, nkv, ps = case["op"], case["nkv"], case["ps"]
    if op == "append":
        n, nq, first = case["n"], case["nq"], case["first"]
        last = first + n if case["one_seq"] else first + 1
        live = torch.zeros(1 if case["one_seq"] else n, (last + ps - 1) // ps, dtype=torch.bool,
                           device="cuda")
        live[:, first // ps:] = True  # the earlier pages belong to the pool too, but are not met
        st["table"], pages = _table(live, g)
        st["k"], st["v"] = _pool(pages, case, g)
        dt = _dt(case["act"])
        st |= dict(q_in=normal(n, nq, HD).to(dt), k_in=normal(n, nkv, HD).to(dt),
                   v_in=normal(n, nkv, HD).to(dt), q_norm=1 + 0.02 * normal(HD),
                   k_norm=1 + 0.02 * normal(HD), rope=_rope(last),
                   q_out=torch.zeros(n, nq, HD, device="cuda", dtype=_dt(case["q"])))
        slots = torch.arange(n, device="cuda", dtype=torch.int32) if case["one_seq"] else \
            torch.zeros(n, device="cuda", dtype=torch.int32)
        st["slots"] = slots + first
        st["pos"] = st["slots"].clone()
        st["seq"] = torch.zeros_like(slots) if case["one_seq"] else None
        if case["plus"]:
            st["q_norm"] -= 1
            st["k_norm"] -= 1
    elif op == "decode":
        B, nq, lens = case["B"], case["nq"], _lens(case)
        live = _live(lens, ps, case["window"], case["sinks"])
        st["table"], pages = _table(live, g)
        st["k"], st["v"] = _pool(pages, case, g)
        st |= dict(lens=i32(lens), q=normal(B, nq, HD),
                   gate=None if case["gate"] == "none" else normal(B, nq, HD).to(_dt(case["gate"])),
                   out=torch.zeros(B, nq, HD, device="cuda", dtype=_dt(case["out"])),
                   sums=normal(B, nkv, live.shape[1] * ps).abs() if case["weights"] else None)
    elif op == "prompt":
        T, s0, nq = case["T"], case["s0"], case["nq"]
        # the pages that some token of the prompt attends to
        span = case["window"] + T - 1 if case["window"] else 0
        st["table"], pages = _table(_live([s0 + T], ps, span, case["sinks"]), g)
        st["k"], st["v"] = _pool(pages, case, g)
        st |= dict(q=normal(T, nq, HD).to(torch.bfloat16),
                   gate=normal(T, nq, HD).to(torch.bfloat16) if case["gate"] else None,
                   out=torch.zeros(T, nq, HD, device="cuda", dtype=torch.bfloat16))
    else:
        B, lens, keep = case["B"], _lens(case), case["keep"]
        live = _live(lens, ps, 0, 0)
        out_pages = (keep + ps - 1) // ps
        st["table"], n_src = _table(live, g)
        dst = torch.randperm(B * out_pages, generator=g, device="cuda").to(torch.int32) + n_src
        st["k"], st["v"] = _pool(n_src + B * out_pages, case, g)
        st["k"][n_src:] = 0
        st["v"][n_src:] = 0
        # sums of weights: most slots got little, a few a lot, some exactly nothing (ties)
        s = torch.rand(B, nkv, live.shape[1] * ps, generator=g, device="cuda") ** 8 * 50
        s[s < 1e-4] = 0
        st |= dict(lens=i32(lens), sums=s, dst=dst.view(B, out_pages), n_src=n_src,
                   new_lens=i32([0] * B), kept=i32([0]).expand(B, nkv, keep).contiguous(),
                   new_sums=torch.zeros(B, nkv, out_pages * ps, device="cuda"))
    return st


# ------------------------------------------------------------------------ plain forms
def _sigmoid(x):
    return 1 / (1 + torch.exp(-x.float()))


def _softmax(s, mask):
    """Softmax over the last dim where mask holds; all zero where it holds nowhere."""
    s = torch.where(mask, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-38)


def _plain_append(st, c):
    def norm_rotate(x, w):
        x = x.float()
        y = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * (w + 1 if c["plus"] else w)
        t = st["rope"][st["pos"].long()][:, None]
        cos, sin, h = t[..., :ROT // 2], t[..., ROT // 2:], ROT // 2
        a, b = y[..., :h], y[..., h:ROT]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., ROT:]], -1)
    slot = st["slots"].long()
    seq = st["seq"].long() if st["seq"] is not None else torch.arange(c["n"], device="cuda")
    page, row = st["table"][seq, slot // c["ps"]].long(), slot % c["ps"]
    k, v = st["k"].clone(), st["v"].clone()
    k[page, :, row] = norm_rotate(st["k_in"], st["k_norm"]).to(k.dtype)
    v[page, :, row] = st["v_in"].to(v.dtype)
    return {"q": norm_rotate(st["q_in"], st["q_norm"]).to(_dt(c["q"])), "k": k, "v": v}


def _plain_decode(st, c):
    B, nq, nkv, n = c["B"], c["nq"], c["nkv"], st["lens"].long()[:, None]
    w = min(c["window"], c["L"])
    if w:  # the sinks before the window, then the window
        i = torch.arange(c["sinks"] + w, device="cuda") - c["sinks"]
        w0 = (n - w).clamp_min(0)
        slot = torch.where(i < 0, i + c["sinks"], w0 + i)
        ok = torch.where(i < 0, slot < w0, slot < n)
    else:
        slot = torch.arange(max(c["L"], 1), device="cuda").expand(B, -1)
        ok = slot < n
    slot = torch.where(ok, slot, 0)
    page = st["table"].long().gather(1, slot // c["ps"]).clamp_min(0)
    k = st["k"][page, :, slot % c["ps"]].float()  # [B][slots][nkv][256]
    v = st["v"][page, :, slot % c["ps"]].float()
    q = st["q"].view(B, nkv, nq // nkv, HD)
    p = _softmax(torch.einsum("bhgd,bshd->bhgs", q, k) / math.sqrt(HD), ok[:, None, None])
    o = torch.einsum("bhgs,bshd->bhgd", p, v).reshape(B, nq, HD)
    if st["gate"] is not None:
        o = o * _sigmoid(st["gate"])
    got = {"out": o.to(_dt(c["out"]))}
    if c["weights"]:
        got["sums"] = st["sums"].scatter_add(2, slot[:, None].expand(-1, nkv, -1),
                                             torch.where(ok[:, None], p.sum(2), 0.0))
    return got


def _plain_prompt(st, c):
    T, s0, nq, nkv, w = c["T"], c["s0"], c["nq"], c["nkv"], c["window"]
    outs = []
    step = max(64, (1 << 24) // (w + 1024 if w else s0 + T))
    for t in range(0, T, step):  # queries in blocks, for the memory that the scores take
        q = st["q"][t:t + step].float().view(-1, nkv, nq // nkv, HD)
        at = s0 + t + torch.arange(len(q), device="cuda")[:, None]
        first = max(s0 + t - w + 1, 0) if w else 0
        slot = torch.arange(first, s0 + t + len(q), device="cuda")
        if w:
            slot = torch.cat([torch.arange(min(c["sinks"], first), device="cuda"), slot])
        page = st["table"][0].long()[slot // c["ps"]]
        k, v = (st[x][page, :, slot % c["ps"]].float() for x in "kv")  # [slots][nkv][256]
        ok = slot <= at
        if w:
            ok = ok & ((slot > at - w) | (slot < c["sinks"]))
        p = _softmax(torch.einsum("thgd,shd->hgts", q, k) / math.sqrt(HD), ok)
        outs.append(torch.einsum("hgts,shd->thgd", p, v).reshape(-1, nq, HD))
    o = torch.cat(outs)
    if st["gate"] is not None:
        o = o * _sigmoid(st["gate"])
    return {"out": o.to(torch.bfloat16)}


def _plain_evict(st, c):
    B, nkv, keep, ps = c["B"], c["nkv"], c["keep"], c["ps"]
    n = st["lens"].long()[:, None, None]
    S = st["sums"].shape[2]
    slot = torch.arange(S, device="cuda").expand(B, nkv, S)
    first, last = slot < c["sinks"], slot >= n - c["recent"]
    rank = torch.where(first | last, math.inf, st["sums"])
    rank = torch.where(slot < n, rank, -math.inf)  # the sums are not negative
    # the keep largest, ties to the lowest slot, in the order of their slots
    order = torch.sort(rank, dim=2, descending=True, stable=True).indices[..., :keep]
    order = torch.where(order < n, order, S).sort(2).values
    order = torch.cat([order, order.new_full((B, nkv, keep - order.shape[2]), S)], 2)
    ok = order < S
    kept = torch.where(ok, order, -1)
    slot = torch.where(ok, order, 0)
    b = torch.arange(B, device="cuda")[:, None, None]
    h = torch.arange(nkv, device="cuda")[None, :, None]
    src = st["table"].long()[b, slot // ps].clamp_min(0)
    j = torch.arange(keep, device="cuda")
    dst = (st["dst"].long() - st["n_src"])[:, j // ps][:, None].expand_as(ok)
    row, head = (j % ps).expand_as(ok), h.expand_as(ok)
    got = {"kept": kept.int(), "lens": st["lens"].clamp_max(keep)}
    for x in "kv":
        got[x] = torch.zeros_like(st[x][st["n_src"]:])
        got[x][dst[ok], head[ok], row[ok]] = st[x][src, head, slot % ps][ok]
    got["sums"] = torch.zeros_like(st["new_sums"])
    got["sums"][..., :keep] = torch.where(ok, st["sums"].gather(2, slot), 0.0)
    return got


# -------------------------------------------------------------------------------- run
def _own_append(st, c):
    from vx27_b200 import ops
    ops.gqa_paged_append(st["q_in"], st["k_in"], st["v_in"], st["q_norm"], st["k_norm"],
                         st["rope"], st["pos"], st["slots"], st["table"], st["k"], st["v"],
                         st["q_out"], seq=st["seq"], eps=EPS, norm_one_plus=c["plus"])
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _own_decode(st, c):
    from vx27_b200 import ops
    if "ws" not in st:  # kept with the caches, for every step
        need = ops.gqa_paged_workspace_bytes(c["B"], c["nq"], c["nkv"], HD,
                                             st["table"].shape[1] * c["ps"], c["window"],
                                             c["sinks"], c["weights"])
        st["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    sums = st["sums"].clone() if c["weights"] else None
    ops.gqa_paged_decode(st["q"], st["gate"], st["k"], st["v"], st["table"], st["lens"], st["out"],
                         st["ws"], window=c["window"], sinks=c["sinks"], weight_sum=sums)
    return {"out": st["out"]} | ({"sums": sums} if c["weights"] else {})


def _own_prompt(st, c):
    from vx27_b200 import ops
    if "ws" not in st:
        need = ops.gqa_paged_prefill_workspace_bytes(c["nkv"], HD)
        st["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    ops.gqa_paged_prefill(st["q"], st["gate"], st["k"], st["v"], st["table"][0], st["out"],
                          s0=c["s0"], window=c["window"], sinks=c["sinks"], workspace=st["ws"])
    return {"out": st["out"]}


def _own_evict(st, c):
    from vx27_b200 import ops
    ops.kv_evict(st["k"], st["v"], st["table"], st["lens"], st["sums"], st["dst"], st["new_lens"],
                 st["new_sums"], st["kept"], c["keep"], sinks=c["sinks"], recent=c["recent"])
    n = st["n_src"]
    return {"kept": st["kept"], "lens": st["new_lens"], "k": st["k"][n:], "v": st["v"][n:],
            "sums": st["new_sums"]}


def run(state):
    c = state["case"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "prompt": _own_prompt,
                "evict": _own_evict}[c["op"]](state, c)
    return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt,
            "evict": _plain_evict}[c["op"]](state, c)


# ----------------------------------------------------------------------- 64-bit values
def _rows(pool, table_row, slots, ps):
    """Rows of the given slots of one sequence, [nkv][slots][256] in 64 bits."""
    flat = pool.transpose(1, 2).reshape(-1, pool.shape[1], HD)
    page = table_row.long().index_select(0, torch.div(slots, ps, rounding_mode="floor"))
    return flat.index_select(0, page * ps + slots % ps).double().transpose(0, 1)


def _attend64(q, k, v, mask):
    """q [nkv][rows][256], k, v [nkv][slots][256], mask [rows][slots] or None: (out, weights)."""
    s = (q.double() / 16) @ k.mT
    if mask is not None:
        s.masked_fill_(~mask, -math.inf)
    p = s.sub_(s.max(-1, keepdim=True).values).exp_()
    p /= p.sum(-1, keepdim=True)
    return p @ v, p


def exact(case, seed):
    st, c, ps = prepare(case, seed), case, case["ps"]
    dev = "cuda"
    if c["op"] == "append":
        def turned(x, w):
            z = x.double()
            z = z / torch.sqrt((z * z).sum(-1, keepdim=True) / HD + EPS)
            z = z * (w.double() + (1.0 if c["plus"] else 0.0))
            ang = st["rope"].double()[st["pos"].long()].unsqueeze(1)
            u = torch.complex(z[..., :32], z[..., 32:64])
            u = u * torch.complex(ang[..., :32].contiguous(), ang[..., 32:].contiguous())
            return torch.cat([u.real, u.imag, z[..., 64:]], -1)
        k, v = st["k"].double(), st["v"].double()
        rows = st["seq"].tolist() if st["seq"] is not None else range(c["n"])
        table, kt, vt = st["table"].tolist(), turned(st["k_in"], st["k_norm"]), st["v_in"].double()
        slots = st["slots"].tolist()
        at = torch.tensor([table[b][s // ps] for b, s in zip(rows, slots)], device=dev)
        off = torch.tensor([s % ps for s in slots], device=dev)
        k.transpose(1, 2)[at, off] = kt
        v.transpose(1, 2)[at, off] = vt
        return {"q": turned(st["q_in"], st["q_norm"]), "k": k, "v": v}
    if c["op"] == "decode":
        nkv, out = c["nkv"], torch.zeros(c["B"], c["nq"], HD, dtype=torch.float64, device=dev)
        sums = st["sums"].double() if c["weights"] else None
        for b, n in enumerate(_lens(c)):
            if not n:
                continue
            lo = max(n - c["window"], 0) if c["window"] else 0
            slots = torch.tensor([*range(min(c["sinks"], lo)), *range(lo, n)], device=dev)
            k, v = (_rows(st[x], st["table"][b], slots, ps) for x in "kv")
            o, p = _attend64(st["q"][b].reshape(nkv, -1, HD), k, v, None)
            out[b] = o.reshape(-1, HD)
            if sums is not None:
                sums[b].index_add_(1, slots, p.sum(1))
        if st["gate"] is not None:
            out *= torch.sigmoid(st["gate"].double())
        return {"out": out} | ({"sums": sums} if c["weights"] else {})
    if c["op"] == "prompt":
        T, s0, nkv, w = c["T"], c["s0"], c["nkv"], c["window"]
        G = c["nq"] // nkv
        out = torch.empty(T, c["nq"], HD, dtype=torch.float64, device=dev)
        for t in range(0, T, 256):
            e = min(T, t + 256)
            lo = max(0, s0 + t + 1 - w) if w else 0
            slots = torch.tensor([*range(min(c["sinks"], lo)), *range(lo, s0 + e)], device=dev)
            k, v = (_rows(st[x], st["table"][0], slots, ps) for x in "kv")
            gap = s0 + torch.arange(t, e, device=dev).repeat(G)[:, None] - slots
            see = (gap >= 0) & ((gap < w) | (slots < c["sinks"]) if w else gap >= 0)
            q = st["q"][t:e].reshape(e - t, nkv, G, HD).permute(1, 2, 0, 3).reshape(nkv, -1, HD)
            o, _ = _attend64(q, k, v, see)
            out[t:e] = o.view(nkv, G, e - t, HD).permute(2, 0, 1, 3).reshape(e - t, -1, HD)
        if st["gate"] is not None:
            out *= torch.sigmoid(st["gate"].double())
        return {"out": out}
    # eviction: whole numbers, and copies of what the kept slots hold
    B, nkv, keep = c["B"], c["nkv"], c["keep"]
    lens, sums = _lens(c), st["sums"].double()
    kept = torch.full((B, nkv, keep), -1, dtype=torch.int32, device=dev)
    k, v = (torch.zeros(st[x][st["n_src"]:].shape, dtype=torch.float64, device=dev) for x in "kv")
    new = torch.zeros(st["new_sums"].shape, dtype=torch.float64, device=dev)
    host = sums.cpu().numpy()
    for b, n in enumerate(lens):
        m = min(n, keep)
        for h in range(nkv):
            if n > keep:
                mid = range(c["sinks"], n - c["recent"])
                best = sorted(mid, key=lambda s: (-host[b, h, s], s))[:keep - c["sinks"] - c["recent"]]
                chosen = [*range(c["sinks"]), *sorted(best), *range(n - c["recent"], n)]
            else:
                chosen = list(range(n))
            if not m:
                continue
            at = torch.tensor(chosen, device=dev)
            kept[b, h, :m] = at.int()
            new[b, h, :m] = sums[b, h, at]
            src = st["table"][b].long()[at // ps]
            j = torch.arange(m, device=dev)
            to = st["dst"][b].long()[j // ps] - st["n_src"]
            k[to, h, j % ps] = st["k"][src, h, at % ps].double()
            v[to, h, j % ps] = st["v"][src, h, at % ps].double()
    return {"kept": kept, "lens": torch.tensor([min(n, keep) for n in lens], dtype=torch.int32,
                                               device=dev), "k": k, "v": v, "sums": new}
