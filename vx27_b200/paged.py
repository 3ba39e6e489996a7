"""A paged BF16 KV cache for the full-attention layers: the pool of pages, the sequences' page
tables and lengths, and what moves pages between them (include/vx27_paged.h). The reference
keeps one contiguous fp32 cache per layer and sequence (src/vx27_qfwd.c:183-185).

All layers of a model hold the same tokens, so one table serves them: page p is a page of
every layer's planes. The tables live on the device; a host copy decides which page goes
where, so nothing is read back. Per sequence the device holds (int32)

    lens   slots held
    pos    positions taken; equal to lens until an eviction cuts the slots back
    step   lens, if the last extend() gave the sequence one token that is no prompt's, else 0 (an
           idle lane of step_paged)

``layer.GQALayer.step_paged`` and ``prompt_paged`` run a layer over it. A round of a server:

    at = cache.extend({0: 1, 1: 1, 5: n}, prompts=[5])   # two running sequences, a new prompt
    for each layer i: step_paged(x, cache, i, ws), prompt_paged(xp, cache, i, 5, *at[5], ws)

A token enters the cache once: by step_paged, or by prompt_paged for the sequences that extend()
was told to be prompts, which matters where a prompt, or its last piece, is one token long.

The tensors keep their addresses, so a captured step_paged may be replayed after each
extend(); extend, release and evict copy from the host and stay outside the capture. All
calls on one cache belong on one stream.
"""
from __future__ import annotations

import torch

from . import ops
from ._lib import Vx27Error


class PagedKV:
    def __init__(self, layers: int, batch: int, n_pages: int, max_pages: int, page_size: int = 64,
                 nkv: int = 4, hd: int = 256, window: int = 0, sinks: int = 0,
                 weights: bool = False, device="cuda"):
        """n_pages pages for batch sequences of at most max_pages pages each. window, sinks: what
        every token attends to (0: everything); pages that fall out of sight are freed. weights:
        the attention each slot gets from the tokens of step_paged is summed, for evict (a
        prompt's tokens add nothing)."""
        if window < 0 or sinks < 0 or (sinks and not window):
            raise Vx27Error(f"PagedKV: window={window} with sinks={sinks}")
        if weights and window:
            raise Vx27Error("PagedKV: eviction keeps slots by their weights, a window by their age: "
                            "one of the two")
        dev = torch.device(device)
        kw = dict(device=dev)
        self.page_size, self.max_pages, self.window, self.sinks = page_size, max_pages, window, sinks
        self.k = torch.empty(layers, n_pages, nkv, page_size, hd, dtype=torch.bfloat16, **kw)
        self.v = torch.empty_like(self.k)
        self.table = torch.full((batch, max_pages), -1, dtype=torch.int32, **kw)
        self._state = torch.zeros(3, batch, dtype=torch.int32, **kw)
        self.lens, self.pos, self.step = self._state
        self.sums = torch.zeros(layers, batch, nkv, max_pages * page_size, **kw) if weights else None
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages = [[-1] * max_pages for _ in range(batch)]
        self._lens, self._pos = [0] * batch, [0] * batch
        self._lanes = set()  # sequences whose token the next step_paged takes

    # ------------------------------------------------------------------ bookkeeping (host)
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._lens[seq]

    def position(self, seq: int) -> int:
        return self._pos[seq]

    def is_lane(self, seq: int) -> bool:
        """Does the sequence's last token go through step_paged?"""
        return seq in self._lanes

    def _check(self, seqs) -> None:
        seqs = list(seqs)
        if len(set(seqs)) != len(seqs) or not all(0 <= s < len(self._lens) for s in seqs):
            raise Vx27Error(f"PagedKV: sequences {seqs} of {len(self._lens)}")

    def _need(self, seq: int, n: int) -> list[int]:
        """Table entries that n more slots of the sequence need a page for."""
        if n < 1:
            raise Vx27Error(f"PagedKV: {n} tokens for sequence {seq}")
        last = self._lens[seq] + n
        if last > self.max_pages * self.page_size:
            raise Vx27Error(f"PagedKV: sequence {seq} holds {self._lens[seq]} slots, {n} more pass "
                            f"{self.max_pages} pages of {self.page_size}")
        return [e for e in range(self._lens[seq] // self.page_size, -(-last // self.page_size))
                if self._pages[seq][e] < 0]

    def _upload(self, seqs) -> None:
        for s in seqs:
            self.table[s].copy_(torch.tensor(self._pages[s], dtype=torch.int32))

    def _upload_state(self, lanes) -> None:
        self._lanes = set(lanes)
        one = [n if s in self._lanes else 0 for s, n in enumerate(self._lens)]
        self._state.copy_(torch.tensor([self._lens, self._pos, one], dtype=torch.int32))

    def _out_of_sight(self, seq: int) -> list[int]:
        """Entries that no later token attends to."""
        if not self.window:
            return []
        ps, lo = self.page_size, self._lens[seq] + 1 - self.window
        first = -(-self.sinks // ps)
        return [e for e in range(first, max(lo, 0) // ps) if self._pages[seq][e] >= 0]

    def extend(self, tokens: dict[int, int], prompts=()) -> dict[int, tuple[int, int]]:
        """Makes room for tokens[seq] more tokens of each sequence and counts them as held:
        (first slot, first position) by sequence. Pages that earlier calls moved out of sight of
        a window are freed first. On the device the state is that after these tokens; a
        sequence that gets one token takes part in the next step_paged, unless it is one of
        prompts, whose tokens go through prompt_paged. The others do not."""
        self._check(tokens)
        prompts = set(prompts)
        if not prompts <= tokens.keys():
            raise Vx27Error(f"PagedKV: prompts {sorted(prompts)} among tokens of {sorted(tokens)}")
        need = {s: self._need(s, n) for s, n in tokens.items()}
        changed = set()
        for s in tokens:
            for e in self._out_of_sight(s):
                self._free.append(self._pages[s][e])
                self._pages[s][e] = -1
                changed.add(s)
        if sum(map(len, need.values())) > len(self._free):
            self._upload(changed)
            raise Vx27Error(f"PagedKV: {sum(map(len, need.values()))} pages needed, "
                            f"{len(self._free)} free")
        at = {}
        for s, n in tokens.items():
            for e in need[s]:
                self._pages[s][e] = self._free.pop()
                changed.add(s)
            at[s] = self._lens[s], self._pos[s]
            self._lens[s] += n
            self._pos[s] += n
        self._upload(changed)
        self._upload_state(s for s, n in tokens.items() if n == 1 and s not in prompts)
        return at

    def release(self, seq: int) -> None:
        """The sequence is done: its pages are free, its lane is idle (the others stay)."""
        self._check([seq])
        self._free += [p for p in self._pages[seq] if p >= 0]
        self._pages[seq] = [-1] * self.max_pages
        self._lens[seq] = self._pos[seq] = 0
        self._upload([seq])
        self._upload_state(self._lanes - {seq})
        if self.sums is not None:
            self.sums[:, seq] = 0

    # --------------------------------------------------------------------------- device
    def evict(self, keep: int, sinks: int = 0, recent: int = 0, seqs=None):
        """Cuts the sequences that hold more than keep slots (all, or those of seqs) back to keep
        of them in every layer and head: the first sinks, the last recent, and those with the
        largest summed weights (vx27_kv_evict). They need ceil(keep / page_size) free pages each
        meanwhile; their old pages are free and their lanes idle afterwards. Returns the sequences
        cut and their kept slots [layers][n][nkv][keep]."""
        if self.sums is None:
            raise Vx27Error("PagedKV: evict needs weights=True")
        seqs = range(len(self._lens)) if seqs is None else list(seqs)
        self._check(seqs)
        if not 0 <= sinks <= sinks + recent <= keep or keep < 1:
            raise Vx27Error(f"PagedKV: keep={keep} with sinks={sinks} and recent={recent}")
        cut = [s for s in seqs if self._lens[s] > keep]
        if not cut:
            return [], None
        n = -(-keep // self.page_size)
        if n * len(cut) > len(self._free):
            raise Vx27Error(f"PagedKV: evict needs {n * len(cut)} free pages, {len(self._free)} are")
        layers, nkv, dev = len(self.k), self.k.shape[2], self.k.device
        # the pages leave the free list, and the sums change, once every layer's call is made
        take = n * len(cut)
        free = self._free[:-take - 1:-1]
        new = [free[i * n:(i + 1) * n] for i in range(len(cut))]
        rows = torch.tensor(cut, device=dev)
        dst = torch.tensor(new, dtype=torch.int32, device=dev)
        table, lens = self.table[rows], self.lens[rows]
        lens_out = torch.empty_like(lens)
        kept = torch.empty(layers, len(cut), nkv, keep, dtype=torch.int32, device=dev)
        out = torch.empty(layers, len(cut), nkv, n * self.page_size, device=dev)
        for i in range(layers):
            ops.kv_evict(self.k[i], self.v[i], table, lens, self.sums[i, rows], dst, lens_out, out[i],
                         kept[i], keep, sinks=sinks, recent=recent)
        del self._free[-take:]
        for j, (s, pages) in enumerate(zip(cut, new)):
            self.sums[:, s] = 0
            self.sums[:, s, :, :n * self.page_size] = out[:, j]
            self._free += [p for p in self._pages[s] if p >= 0]
            self._pages[s] = pages + [-1] * (self.max_pages - n)
            self._lens[s] = keep
        self._upload(cut)
        self._upload_state(self._lanes - set(cut))
        return cut, kept

    def workspace(self, nq: int) -> torch.Tensor:
        """Scratch for decode and prompt calls over this cache (one stream's at a time)."""
        nkv, hd = self.k.shape[2], self.k.shape[4]
        need = max(ops.gqa_paged_workspace_bytes(len(self._lens), nq, nkv, hd,
                                                 self.max_pages * self.page_size, self.window,
                                                 self.sinks, self.sums is not None),
                   ops.gqa_paged_prefill_workspace_bytes(nkv, hd))
        return torch.empty(need, dtype=torch.uint8, device=self.k.device)
