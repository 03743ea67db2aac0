"""Ops over a page pool that streams share: attention of a step's rows whose streams have a long prefix in common, the weight that the rows gave to every
cached key, and eviction by it. `TorchShared` states them in plain fp32 PyTorch (the oracle of the GPU tests and the CPU path); `CudaShared` calls the
kernels of `csrc/shared_attn.cu`, `csrc/kv_mass.cu` and `csrc/kv_evict.cu`. Both are mixed into the op classes (`TorchOps`, `CudaOps`).

A step's rows come in segments of one slot each, `segs` = (seg_slot, seg_row0, seg_nrows, rows of the longest): rows seg_row0 .. seg_row0 + seg_nrows, in any
order; row i sees the first row_kvlen[i] tokens. `groups` = (grp_seg0, grp_nsegs, grp_len), or None: the rows of grp_nsegs consecutive segments from grp_seg0
on lie side by side and read their first grp_len tokens, any number, through the table of the first of these segments, and what follows through their
own (whose entries for whole shared pages are not looked at). A segment belongs to one group at most; one of no rows is padding, whatever its slot (but that of
a group's first; inside a group it lies between the rows of its neighbours). Streams whose tables hold the same pages (a pool whose owner lets several streams
have a page: samples of one prompt, forks of one conversation) are a group, so that their common keys and values are read once for every 128 (row, head) pairs
of it. A row is of one segment; of none, it is left out and its output says nothing. Caches are [pages, kv_block, kv heads, head dim] in bf16, kv_block a
multiple of 64. What the kernels find wrong in the tables on the device (a page or slot that is none, a context beyond its table, a segment of more rows than
was said) sets the op class's status word.

Where contexts are cut follows the lengths of the whole step: a row may round otherwise beside other streams, decoded or verified, than by itself (the paged
attention of every stream by itself does not). The same call gives the same bits. A call plans 5 words a segment, 4 a group and 2 a block of rows (128 pairs of a row
and a query head of one kv head for the attention, 64 for the sums), 40960 in all, and is refused beyond: from about 20000 rows on where 128 query heads share a kv
head, 320000 where 8 do (160000 for the sums), half as many in groups.

Sums of weights are [pages, kv heads, kv_block] in fp32, beside the cache: they follow the pages through forks and parking. Whoever writes a key into a page sets its sum,
to zero or what it is to start from: the ops change the sums of keys that a step sees and of places that tokens are moved to, and leave those behind a page's last token, a
former owner's among them, as they are.
"""
from __future__ import annotations

import math

import torch


def _spans(segs, groups):
    """(segment, slot that the shared tokens are read through, shared tokens, group or -1) of every segment."""
    out = []
    for s in range(len(segs[0])):
        slot, shared, group = int(segs[0][s]), 0, -1
        for g in range(0 if groups is None else len(groups[0])):
            lo = int(groups[0][g])
            if lo <= s < lo + int(groups[1][g]):
                slot, shared, group = int(segs[0][lo]), int(groups[2][g]), g
        out.append((s, slot, shared, group))
    return out


def _token_rows(block_table, kv_block, slot, shared_slot, shared, n):
    """Numbers of the cache rows of the first n tokens."""
    pos = torch.arange(n, device=block_table.device)
    at = torch.where(pos < shared, block_table[shared_slot, pos // kv_block], block_table[slot, pos // kv_block]).long()
    return at * kv_block + pos % kv_block


class TorchShared:
    def attention_shared(self, q, proj, k_cache, v_cache, row_kvlen, block_table, kv_block, nq, nkv, hd, gated, segs, groups=None, want_lse=False):
        """o = softmax(q k / sqrt(hd)) v over what a row sees, [rows, nq * hd]; zeros where it sees nothing. With `want_lse` also the natural
        logarithm of the softmax's sum, fp32 [rows, nq] (-inf where a row sees nothing)."""
        T = q.shape[0]
        out = torch.zeros(T, nq, hd, dtype=torch.float32, device=q.device)
        lse = torch.full((T, nq), -math.inf, dtype=torch.float32, device=q.device)
        kf, vf = k_cache.reshape(-1, nkv, hd), v_cache.reshape(-1, nkv, hd)
        for s, shared_slot, shared, _ in _spans(segs, groups):
            for t in range(int(segs[1][s]), int(segs[1][s]) + int(segs[2][s])):
                n = int(row_kvlen[t])
                if n <= 0:
                    continue
                at = _token_rows(block_table, kv_block, int(segs[0][s]), shared_slot, shared, n)
                x = torch.einsum("kgd,tkd->kgt", q[t].reshape(nkv, -1, hd).float(), kf[at].float()) / math.sqrt(hd)
                out[t] = torch.einsum("kgt,tkd->kgd", torch.softmax(x, -1), vf[at].float()).reshape(nq, hd)
                lse[t] = torch.logsumexp(x, -1).reshape(nq)
        if gated:
            out = out * torch.sigmoid(proj[:, :nq * 2 * hd].float().view(T, nq, 2 * hd)[..., hd:])
        out = out.reshape(T, nq * hd).to(self.dtype)
        return (out, lse) if want_lse else out

    def attention_mass(self, q, k_cache, mass, row_kvlen, block_table, kv_block, nq, nkv, hd, segs, groups=None, lse=None, carry=1.0, out=None):
        """Per kv head and key that some row sees: out = carry * mass + the sum of exp(q k / sqrt(hd) - lse) over the rows that see the key and the heads
        that share the kv head (64 at most); `out` is `mass` itself unless given, other entries stay. `lse` is that of the step's attention, or None: it
        is computed. With carry 0 `mass` is not read. A key is of one segment, or of one group's shared tokens: one that two of them hold is an error (of streams
        that were forked at different tokens; a call for each of them, with carry 1, adds their weights up)."""
        out = mass if out is None else out
        kf = k_cache.reshape(-1, nkv, hd)
        sums = torch.zeros(mass.shape[0] * kv_block, nkv, dtype=torch.float32, device=q.device)
        seen = torch.zeros(sums.shape[0], dtype=torch.bool, device=q.device)
        holder = torch.full((sums.shape[0],), -1, dtype=torch.int64, device=q.device)
        for s, shared_slot, shared, group in _spans(segs, groups):
            rows = range(int(segs[1][s]), int(segs[1][s]) + int(segs[2][s]))
            longest = max([int(row_kvlen[t]) for t in rows] + [0])
            if longest <= 0:
                continue
            at = _token_rows(block_table, kv_block, int(segs[0][s]), shared_slot, shared, longest)
            seen[at] = True
            for part, who in ((at[:max(shared, 0)], group), (at[max(shared, 0):], -2 - s)):
                if part.unique().numel() < part.numel() or not ((holder[part] == -1) | (holder[part] == who)).all():
                    raise RuntimeError("attention_mass: a key of two segments, or of a segment and a group's shared tokens")
                holder[part] = who
            for t in rows:
                n = int(row_kvlen[t])
                if n <= 0:
                    continue
                x = torch.einsum("kgd,tkd->kgt", q[t].reshape(nkv, -1, hd).float(), kf[at[:n]].float()) / math.sqrt(hd)
                l = torch.logsumexp(x, -1) if lse is None else lse[t].reshape(nkv, -1).float()
                sums.index_add_(0, at[:n], torch.exp(x - l[..., None]).sum(1).t())
        new = sums.view(-1, kv_block, nkv).transpose(1, 2)
        new = new + carry * mass if carry else new
        out.copy_(torch.where(seen.view(-1, 1, kv_block), new, out))
        return out

    def kv_evict(self, k_cache, v_cache, kv_scale, mass, seg_slot, seg_len, block_table, dst_table, kv_block, keep, first=0, recent=0):
        """Per slot of `seg_slot` (with seg_len tokens) and kv head, `keep` tokens move to the pages dst_table[segment], in their order: the `first` first
        ones, the `recent` last ones, and of the others those with the largest sums (the earlier of equal ones; a sum that is no number counts as the
        largest). Keys, values, scales and sums are copied; contexts of up to `keep` tokens whole. The new pages are none of the old ones; places of theirs
        behind the last token kept stay as they were, sums too. Returns the tokens kept, int32 [segments, kv heads, keep], ascending, -1 behind the last.
        Caches of codes move as they are, with sums that their owner has: `attention_mass` reads bf16 caches."""
        nkv = k_cache.shape[2]
        if not 0 <= first <= keep - recent <= keep or keep < 1 or dst_table.shape[1] * kv_block < keep:
            raise RuntimeError(f"kv_evict: first {first} and recent {recent} of {keep}, pages for {dst_table.shape[1] * kv_block}")
        kept = torch.full((len(seg_slot), nkv, keep), -1, dtype=torch.int32, device=k_cache.device)
        for s in range(len(seg_slot)):
            slot, n = int(seg_slot[s]), int(seg_len[s])
            pos = torch.arange(max(n, keep), device=k_cache.device)
            src_page, to_page = block_table[slot, pos[:n] // kv_block].long(), dst_table[s, pos[:keep] // kv_block].long()
            for h in range(nkv):
                ids = pos[:n]
                if n > keep:
                    w = mass[src_page, h, ids % kv_block][first:n - recent]
                    best = torch.sort(w, descending=True, stable=True).indices[:keep - first - recent] + first
                    ids = torch.cat([pos[:first], best.sort().values, pos[n - recent:n]])
                m = len(ids)
                kept[s, h, :m] = ids.int()
                a, b, c, d = src_page[ids], ids % kv_block, to_page[:m], pos[:m] % kv_block
                for x in (k_cache, v_cache, kv_scale):
                    if x is not None:
                        x[c, d, h] = x[a, b, h]
                mass[c, h, d] = mass[a, h, b]
        return kept


class CudaShared:
    def _shared_step(self, q, nq, hd, segs, groups):
        """Queries as the kernels read them ([rows, nq, hd], rows any multiple of 16 bytes apart) and the step's tables as arguments."""
        q = q.view(q.shape[0], nq, hd) if q.dim() == 2 else q
        if q.stride(-1) != 1 or q.stride(1) != hd or (q.shape[0] > 1 and q.stride(0) % 8) or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
        return q, (*segs, *(groups if groups is not None else (None, None, None)))

    def attention_shared(self, q, proj, k_cache, v_cache, row_kvlen, block_table, kv_block, nq, nkv, hd, gated, segs, groups=None, want_lse=False):
        """Attention of a step's rows over a cache whose streams share pages; the oracle's docstring and the top of this file say what of. `proj` is read
        for the output gate only. It takes less time than the paged attention of every stream by itself from about 4 streams of 1024 shared tokens on, or 2 of
        4096 (24 query heads of 256 columns over 4; 32 of 128 over 8: 16 of 1024, 4 of 4096, 2 of 16000): at 32 of 16000 55 us instead of 529. Below that,
        and for up to four streams without groups, it takes up to 8 us more."""
        if gated and proj is None:
            raise RuntimeError("attention_shared: no proj to gate with")
        q, step = self._shared_step(q, nq, hd, segs, groups)
        T, G = q.shape[0], 0 if groups is None else groups[0].numel()
        out = self.empty(T, nq * hd, dtype=torch.bfloat16, device=q.device)
        lse = self.empty(T, nq, dtype=torch.float32, device=q.device) if want_lse else None
        ws = self.empty(self.C.attention_shared_floats(T, segs[0].numel(), segs[3], G, nq, nkv, hd, self.sm_count, 1), dtype=torch.float32, device=q.device)
        self.launches += 2 if T and segs[0].numel() else 0
        self.C.attention_shared(out, lse, ws, q, k_cache, v_cache, proj if gated else None, row_kvlen, block_table, kv_block, nq, nkv, hd, *step,
                                self.sm_count, self.status_word)
        return (out, lse) if want_lse else out

    def attention_mass(self, q, k_cache, mass, row_kvlen, block_table, kv_block, nq, nkv, hd, segs, groups=None, lse=None, carry=1.0, out=None):
        """Weight that the step's rows gave to every key of their contexts, added to `carry` times the sums so far (see the oracle). A key that
        two segments hold, or a segment and a group's shared tokens, sets the status, and its sum says nothing."""
        q, step = self._shared_step(q, nq, hd, segs, groups)
        out = mass if out is None else out
        G = 0 if groups is None else groups[0].numel()
        ws = self.empty(self.C.attention_mass_floats(q.shape[0], segs[0].numel(), segs[3], G, nq, nkv, hd, block_table.shape[1] * kv_block,
                                                     k_cache.shape[0] * kv_block, lse is None, self.sm_count), dtype=torch.float32, device=q.device)
        self.launches += self.C.attention_mass(out, mass, float(carry), lse, ws, q, k_cache, row_kvlen, block_table, kv_block, nq, nkv, hd, *step,
                                               self.sm_count, self.status_word)
        return out

    def kv_evict(self, k_cache, v_cache, kv_scale, mass, seg_slot, seg_len, block_table, dst_table, kv_block, keep, first=0, recent=0):
        """Eviction by accumulated weight into new pages (see the oracle); rows of every cache form move as they are."""
        kept = self.empty(seg_slot.numel(), k_cache.shape[2], keep, dtype=torch.int32, device=k_cache.device)
        self.launches += 2 if seg_slot.numel() else 0
        self.C.kv_evict(kept, k_cache, v_cache, kv_scale, mass, seg_slot, seg_len, block_table, dst_table, kv_block, keep, first, recent,
                        self.sm_count, self.status_word)
        return kept
