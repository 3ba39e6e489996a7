"""The paged cache's entry points refuse bad arguments before anything is launched (no GPU
needed: the C checks see only numbers and pointers, the wrappers only shapes and types)."""
import ctypes as C

import pytest
import torch

from vx27_b200 import ops

P = C.c_void_p
HD = 256


def _call(vxlib, name, args):
    err = C.create_string_buffer(256)
    rc = getattr(vxlib, name)(*args, None, err, 256)
    return rc, err.value.decode()


def _append(**o):
    a = dict(q=P(16), k=P(16), v=P(16), qw=P(16), kw=P(16), rope=P(16), rl=64, pos=P(4), slots=P(4),
             seq=None, table=P(4), ns=2, mp=4, kp=P(16), vp=P(16), n_pages=8, ps=16, qo=P(16), n=2,
             nq=24, nkv=4, hd=HD, rd=64, eps=1e-6, flags=0)
    a.update(o)
    return list(a.values())


def _decode(**o):
    a = dict(q=P(16), gate=None, kp=P(16), vp=P(16), n_pages=8, ps=16, table=P(4), mp=4, lens=P(4),
             window=0, sinks=0, wsum=None, out=P(16), ws=P(16), wsb=1 << 30, B=2, nq=24, nkv=4,
             hd=HD, splits=0, flags=0)
    a.update(o)
    return list(a.values())


def _prefill(**o):
    a = dict(q=P(16), gate=None, kp=P(16), vp=P(16), n_pages=8, ps=16, table=P(4), mp=4, s0=0,
             window=0, sinks=0, out=P(16), ws=P(16), wsb=1 << 30, T=8, nq=24, nkv=4, hd=HD, flags=3)
    a.update(o)
    return list(a.values())


def _evict(**o):
    a = dict(kp=P(16), vp=P(32), n_pages=8, ps=16, table=P(4), mp=4, lens=P(4), ws=P(16),
             table2=P(8), mp2=2, lens2=P(8), ws2=P(8), kept=P(4), keep=20, sinks=4, recent=8, B=2,
             nkv=4, hd=HD)
    a.update(o)
    return list(a.values())


POOL = [(dict(hd=128), "hd=128"), (dict(ps=48), "page_size=48"), (dict(ps=8), "page_size=8"),
        (dict(ps=512), "page_size=512"), (dict(n_pages=0), "bad shape"), (dict(mp=0), "bad shape"),
        (dict(kp=None), "null pointer"), (dict(table=None), "null pointer"),
        (dict(kp=P(8)), "16-byte aligned"), (dict(nkv=0), "nkv=0"),
        (dict(n_pages=1 << 26), "over 2\\^31 rows"), (dict(mp=1 << 28), "over 2\\^31 rows")]
HEADS = [(dict(nq=36), "1 to 8 query heads"), (dict(nq=25), "1 to 8 query heads"),
         (dict(nq=0), "1 to 8 query heads")]
WINDOW = [(dict(window=-1), "window=-1"), (dict(window=4, sinks=-1), "sinks=-1"),
          (dict(sinks=4), "sinks need a window")]


@pytest.mark.parametrize("name,make,cases", [
    ("vx27_gqa_paged_append", _append, POOL + HEADS + [
        (dict(n=0), "n=0"), (dict(n=3), "3 tokens for 2 sequences"), (dict(rd=24), "rope_dim=24"),
        (dict(rd=272), "rope_dim=272"), (dict(rope=None), "null pointer"),
        (dict(q=P(8)), "16-byte aligned"), (dict(slots=None), "null pointer")]),
    ("vx27_gqa_paged_decode", _decode, POOL + HEADS + WINDOW + [
        (dict(B=0), "B=0"), (dict(B=65536), "B=65536"), (dict(lens=None), "null pointer"),
        (dict(wsum=P(8)), "16-byte aligned"),
        (dict(ws=None), "null pointer"), (dict(wsb=0), "workspace of 0 bytes"),
        (dict(out=P(24)), "16-byte aligned")]),
    ("vx27_gqa_paged_prefill", _prefill, POOL + HEADS + WINDOW + [
        (dict(flags=1), "must be bf16"), (dict(flags=2), "must be bf16"), (dict(T=0), "slots"),
        (dict(T=65), "slots \\[0, 0 \\+ 65\\)"), (dict(s0=-1), "slots"),
        (dict(s0=0x7ffffff0, T=64), "slots"), (dict(wsb=100), "workspace of 100 bytes")]),
    ("vx27_kv_evict", _evict, POOL + [
        (dict(B=0), "B=0"), (dict(keep=0), "keep=0"), (dict(recent=17), "keep=20"),
        (dict(sinks=-1), "keep=20"), (dict(sinks=0x7fffffff, recent=0x7fffffff), "keep=20"),
        (dict(mp2=1), "1 pages"), (dict(mp2=0), "0 pages"), (dict(ws=None), "null pointer"),
        (dict(table2=P(4)), "an output is an input"), (dict(lens2=P(4)), "an output is an input"),
        (dict(ws2=P(16)), "an output is an input"), (dict(ws=P(20)), "16-byte aligned"), (dict(vp=P(16)), "an output is an input")]),
])
def test_c_refusals(vxlib, name, make, cases):
    import re
    for change, message in cases:
        rc, err = _call(vxlib, name, make(**change))
        assert rc == -1 and re.search(message, err), (name, change, rc, err)


def test_workspace_sizes(vxlib):
    assert ops.gqa_paged_prefill_workspace_bytes(0, HD) == 0
    assert 2 * 4 * 64 * 512 < ops.gqa_paged_prefill_workspace_bytes(4, HD) < 64 << 20
    assert ops.gqa_paged_workspace_bytes(0, 24, 4, HD, 64) == 0
    big = ops.gqa_paged_workspace_bytes(64, 24, 4, HD, 4096, weights=True)
    assert 0 < ops.gqa_paged_workspace_bytes(1, 24, 4, HD, 64) <= big < 1 << 31


def test_wrapper_refusals():
    E = ops.Vx27Error
    B, nq, nkv, ps, mp = 2, 24, 4, 16, 4
    bf = torch.bfloat16
    kp = torch.zeros(8, nkv, ps, HD, dtype=bf)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    q, out, ws = torch.zeros(B, nq, HD), torch.zeros(B, nq, HD), torch.zeros(64)
    dec = lambda **o: ops.gqa_paged_decode(**(dict(  # noqa: E731
        q=q, gate=None, k_pages=kp, v_pages=kp, page_table=i(B, mp), lens=i(B), out=out,
        workspace=ws) | o))
    for change, message in [
            (dict(k_pages=kp.float()), "k_pages: dtype"), (dict(v_pages=kp[:4]), "v_pages: shape"),
            (dict(q=q.to(bf)), "q: dtype"), (dict(gate=q[:1]), "gate: shape"),
            (dict(page_table=i(B + 1, mp)), "page_table: shape"),
            (dict(page_table=i(B, mp).long()), "page_table: dtype"),
            (dict(lens=i(B + 1)), "lens: shape"), (dict(out=out.double()), "out: dtype"),
            (dict(weight_sum=torch.zeros(B, nkv, 8)), "weight_sum: shape"),
            (dict(), "expected a contiguous CUDA tensor")]:
        with pytest.raises(E, match=message):
            dec(**change)
    n = 3
    x, kv = torch.zeros(n, nq, HD, dtype=bf), torch.zeros(n, nkv, HD, dtype=bf)
    app = lambda **o: ops.gqa_paged_append(**(dict(  # noqa: E731
        q_in=x, k_in=kv, v_in=kv, q_norm_w=torch.zeros(HD), k_norm_w=torch.zeros(HD),
        rope=torch.zeros(8, 64), pos=i(n), slots=i(n), page_table=i(n, mp), k_pages=kp, v_pages=kp,
        q_out=x) | o))
    for change, message in [
            (dict(k_in=kv.float()), "k_in: dtype"), (dict(v_in=kv[:, :2]), "v_in: shape"),
            (dict(pos=i(n + 1)), "pos: shape"), (dict(seq=i(n).long()), "seq: dtype"),
            (dict(q_out=x.half()), "q_out: dtype"), (dict(rope=torch.zeros(64)), "rope: shape"),
            (dict(q_norm_w=torch.zeros(8)), "q_norm_w: shape"),
            (dict(page_table=i(mp)), "page_table: shape")]:
        with pytest.raises(E, match=message):
            app(**change)
    y = torch.zeros(n, nq, HD, dtype=bf)
    pre = lambda **o: ops.gqa_paged_prefill(**(dict(  # noqa: E731
        q=x, gate=None, k_pages=kp, v_pages=kp, page_table=i(mp), out=y, workspace=ws) | o))
    for change, message in [
            (dict(q=x.float()), "q: dtype"), (dict(gate=x.float()), "gate: dtype"),
            (dict(out=y.float()), "out: dtype"), (dict(page_table=i(1, mp)), "page_table: shape")]:
        with pytest.raises(E, match=message):
            pre(**change)
    ev = lambda **o: ops.kv_evict(**(dict(  # noqa: E731
        k_pages=kp, v_pages=kp, page_table=i(B, mp), lens=i(B),
        weight_sum=torch.zeros(B, nkv, mp * ps), page_table_out=i(B, 2), lens_out=i(B),
        weight_sum_out=torch.zeros(B, nkv, 2 * ps), kept=i(B, nkv, 20), keep=20) | o))
    for change, message in [
            (dict(weight_sum=torch.zeros(B, nkv, ps)), "weight_sum: shape"),
            (dict(weight_sum_out=torch.zeros(B, nkv, ps)), "weight_sum_out: shape"),
            (dict(kept=i(B, nkv, 21)), "kept: shape"), (dict(lens_out=i(1)), "lens_out: shape"),
            (dict(page_table_out=i(1, 2)), "page_table_out: shape")]:
        with pytest.raises(E, match=message):
            ev(**change)


def cache(**o):
    from vx27_b200.paged import PagedKV
    return PagedKV(**(dict(layers=2, batch=3, n_pages=10, max_pages=4, page_size=16, nkv=1,
                           device="cpu") | o))


def held(c):
    """Pages that the tables name, checked against the host's copy and the free list."""
    pages = [p for row in c.table.tolist() for p in row if p >= 0]
    assert c.table.tolist() == c._pages
    assert c.lens.tolist() == c._lens and c.pos.tolist() == c._pos
    assert all(a in (0, b) for a, b in zip(c.step.tolist(), c._lens))
    assert len(set(pages)) == len(pages) and sorted(pages + c._free) == list(range(len(c.k[0])))
    return pages


def test_paged_cache_hands_out_and_takes_back_pages():
    c = cache()
    assert c.extend({0: 17, 2: 16}) == {0: (0, 0), 2: (0, 0)}
    assert len(held(c)) == 3 and c.lens.tolist() == [17, 0, 16] and c.free_pages == 7
    assert c.extend({0: 15}) == {0: (17, 17)} and len(held(c)) == 3
    assert c.extend({0: 1, 1: 1, 2: 33}) == {0: (32, 32), 1: (0, 0), 2: (16, 16)}
    assert len(held(c)) == 8 and c.step.tolist() == [33, 1, 0]
    with pytest.raises(ops.Vx27Error, match="3 pages needed, 2 free"):
        c.extend({1: 60})
    with pytest.raises(ops.Vx27Error, match="pass 4 pages of 16"):
        c.extend({1: 1, 2: 16})
    with pytest.raises(ops.Vx27Error, match="0 tokens"):
        c.extend({1: 0})
    assert len(held(c)) == 8 and c.lens.tolist() == [33, 1, 49]
    for seqs in ({3: 1}, {-1: 1}):
        with pytest.raises(ops.Vx27Error, match="sequences"):
            c.extend(seqs)
    with pytest.raises(ops.Vx27Error, match="sequences"):
        c.release(-1)
    c.release(2)
    assert len(held(c)) == 4 and c.length(2) == c.position(2) == 0
    c.extend({1: 60})
    assert len(held(c)) == 7


def test_paged_cache_frees_what_a_window_leaves():
    c = cache(n_pages=6, max_pages=100, window=20, sinks=3)
    total = 0
    for n in (40, 1, 1, 30, 1, 500 - 73, 1):
        if n > 60:  # more at once than the pages hold
            with pytest.raises(ops.Vx27Error, match="free"):
                c.extend({1: n})
            continue
        c.extend({1: n})
        total += n
        held(c)
        have = [e for e, p in enumerate(c._pages[1]) if p >= 0]
        # what the first of the new tokens saw, to the end, and the sinks
        seen = {j // 16 for j in range(total) if j < 3 or j > total - n - 20}
        assert set(have) == seen, (total, have, seen)
    assert c.length(1) == c.position(1) == total


def test_paged_cache_refusals():
    with pytest.raises(ops.Vx27Error, match="one of the two"):
        cache(window=4, weights=True)
    for window, sinks in ((-1, 0), (4, -1), (0, 2)):
        with pytest.raises(ops.Vx27Error, match="window="):
            cache(window=window, sinks=sinks)
    c = cache()
    with pytest.raises(ops.Vx27Error, match="weights=True"):
        c.evict(4)
    c = cache(weights=True)
    assert c.evict(4) == ([], None)
    c.extend({0: 64, 1: 60})
    with pytest.raises(ops.Vx27Error, match="evict needs 4 free pages"):
        c.evict(20)
    with pytest.raises(ops.Vx27Error, match="keep=8"):
        c.evict(8, sinks=4, recent=5)
    for bad in ([1, 1], [-1], [3]):
        with pytest.raises(ops.Vx27Error, match="sequences"):
            c.evict(20, seqs=bad)
    held(c)


def test_layer_refuses_a_prompt_without_room():
    from vx27_b200.layer import GQALayer
    layer, c = object.__new__(GQALayer), cache()
    c.extend({1: 20})
    for seq, slot, n in ((1, 0, 21), (1, 15, 6), (1, -1, 5), (0, 0, 1), (-1, 0, 1)):
        with pytest.raises(ops.Vx27Error, match="prompt_paged"):
            layer.prompt_paged(torch.zeros(n, 8), c, 0, seq, slot, slot, None)


@pytest.mark.parametrize("fails", ["kept", 0, 1])
def test_an_eviction_that_fails_changes_nothing(monkeypatch, fails):
    """Memory that runs out before the first layer, or a call refused in a layer: pages, tables,
    lengths and sums stay as they were, and the eviction succeeds when called again."""
    from vx27_b200 import paged
    c = cache(weights=True, n_pages=12)
    c.extend({0: 60, 2: 33})
    c.extend({1: 1})
    c.sums.copy_(torch.rand(c.sums.shape))
    sums, free = c.sums.clone(), list(c._free)
    calls = []

    def kv_evict(k, v, table, lens, s, table_out, lens_out, s_out, kept, keep, sinks, recent):
        if broken and len(calls) == fails:
            raise ops.Vx27Error("refused")
        calls.append(table_out.tolist())
        lens_out.fill_(keep)
        s_out.fill_(7)
        kept.fill_(len(calls))

    def empty(*shape, **kw):
        if broken and fails == "kept":
            raise torch.OutOfMemoryError("no memory")
        return make(*shape, **kw)
    make, broken = torch.empty, True
    monkeypatch.setattr(paged.ops, "kv_evict", kv_evict)
    monkeypatch.setattr(paged.torch, "empty", empty)
    with pytest.raises((ops.Vx27Error, torch.OutOfMemoryError)):
        c.evict(20, sinks=2, recent=4)
    assert c._free == free and torch.equal(c.sums, sums) and c._lens == [60, 1, 33]
    held(c)
    broken = False
    calls.clear()
    cut, kept = c.evict(20, sinks=2, recent=4)
    assert cut == [0, 2] and kept[:, 0, 0, 0].tolist() == [1, 2]
    assert c._lens == [20, 1, 20] and len(held(c)) == 5
    assert all(t == [c._pages[0][:2], c._pages[2][:2]] for t in calls) and len(calls) == 2
    for s in (0, 2):
        assert (c.sums[:, s, :, :32] == 7).all() and (c.sums[:, s, :, 32:] == 0).all()
    assert torch.equal(c.sums[:, 1], sums[:, 1])


def test_a_prompt_of_one_token_is_no_lane():
    """extend(prompts=...): the device's step entry stays 0 for a prompt's single token, and
    prompt_paged refuses a token that is a lane of step_paged, which would store it a second time."""
    from vx27_b200.layer import GQALayer
    layer, c = object.__new__(GQALayer), cache()
    c.extend({0: 5, 1: 20})
    c.extend({0: 1, 1: 1, 2: 1}, prompts=[1, 2])
    assert c.step.tolist() == [6, 0, 0]
    held(c)
    with pytest.raises(ops.Vx27Error, match="lane of step_paged"):
        layer.prompt_paged(torch.zeros(1, 8), c, 0, 0, 5, 5, None)
    with pytest.raises(ops.Vx27Error, match="lane of step_paged"):
        layer.prompt_paged(torch.zeros(3, 8), c, 0, 0, 3, 3, None)
    before = c._lens[:]
    for prompts in ([1], [3], [-1], [0, 2]):
        with pytest.raises(ops.Vx27Error, match="prompts"):
            c.extend({0: 1, 2: 3} if prompts != [0, 2] else {0: 1}, prompts=prompts)
    assert c._lens == before and c.step.tolist() == [6, 0, 0]

    class Reached(Exception):
        pass

    def project(*a):
        raise Reached
    layer._project = project
    for seq, slot, n in ((1, 20, 1), (1, 0, 21), (2, 0, 1), (0, 0, 5)):  # prompts, earlier slots
        with pytest.raises(Reached):
            layer.prompt_paged(torch.zeros(n, 8), c, 0, seq, slot, slot, None)
    c.extend({2: 4})  # a later call's lanes alone count
    with pytest.raises(Reached):
        layer.prompt_paged(torch.zeros(1, 8), c, 0, 0, 5, 5, None)


def test_lanes_outlive_what_happens_to_other_sequences(monkeypatch):
    """release and evict between extend and step_paged idle the sequences that they change, and
    leave the others' lanes."""
    from vx27_b200 import paged
    c = cache(weights=True, batch=4, n_pages=20)
    c.extend({0: 3, 1: 40, 2: 50, 3: 3})
    c.extend({0: 1, 1: 1, 2: 1, 3: 1}, prompts=[3])
    assert c.step.tolist() == [4, 41, 51, 0]
    c.release(1)
    assert c.step.tolist() == [4, 0, 51, 0] and c.is_lane(0) and not c.is_lane(1)
    monkeypatch.setattr(paged.ops, "kv_evict", lambda *a, **kw: None)
    assert c.evict(20)[0] == [2]
    assert c.step.tolist() == [4, 0, 0, 0] and c.is_lane(0) and not c.is_lane(2)
    held(c)
