"""Paged state-tree KV cache: keys and values stored losslessly in 16-token pages of state-tree records (6400 B per
page per KV head against 8192 B in BF16), appended on write and read by the decode attention kernel without ever
being expanded.  PageStore holds one attention layer's pages (the tensors of the reference's statetree/kvcache.py
StateTreeKVLayer 49-57, with its append / dense / attention calls); PageStore8 holds them in 8 bits (no counterpart in the
reference); PagedKVCache is the static cache of the decode runner in this package.  The Hugging Face classes of the reference (StateTreeKVCache, StateTreeKVLayer,
statetree_attention, enable) live in hf_cache.py and are re-exported here when transformers is importable.
"""
import torch

from .ops import calls, kv_ext, lib

PAGE = 16
RKV = 1600


def decode_splits(B, Hkv, max_pages, sms=148, min_pages=4):
    """How many CTAs share each (sequence, KV head) of the decode attention kernel.  Two bounds: the split that
    balances a split's own pages against the cost of merging the partial results grows like the square root of the
    page count, and no more splits are needed than fill the GPU about three CTAs deep.  At least min_pages pages
    per split.  A function of the batch size and the longest context only, so one captured graph per batch size
    serves every step (the role of the reference's statetree/vllm_kv.py:42-50, re-sized for 148 SMs)."""
    by_length = int(round(max_pages ** 0.5))
    by_fill = -(-3 * sms // max(1, B * Hkv))
    most = max(1, max_pages // max(1, min_pages))
    return min(most, max(2, min(by_length, by_fill, 64)))               # two splits at least: several waves of CTAs


class PageStore:
    """pages of one attention layer: uint8 [blocks, H, 2, 2, 1600], escape pool int32 [P, 16], pool counter int32 [2]"""

    def __init__(self, num_blocks, num_kv_heads, device, pool_blocks=1 << 15):
        self._take(torch.zeros(num_blocks, num_kv_heads, 2, 2, RKV, dtype=torch.uint8, device=device),
                   torch.zeros(pool_blocks, 16, dtype=torch.int32, device=device), torch.zeros(2, dtype=torch.int32, device=device))

    @classmethod
    def over(cls, pages, pool, pcnt=None):
        """a store over tensors that exist already (another store's, part of a larger buffer, pages that were saved).  pcnt: the pool's
        counter, for appends; None: every block of the pool counts as taken"""
        self = cls.__new__(cls)
        kv_ext()._pages("PageStore", pages, pool, pcnt)
        if pcnt is None:
            pcnt = torch.tensor([pool.shape[0], 0], dtype=torch.int32, device=pages.device)
        if pcnt.dtype != torch.int32 or pcnt.numel() != 2:
            raise RuntimeError("PageStore: pool counter int32 [2]")
        self._take(pages, pool, pcnt)
        return self

    def _take(self, pages, pool, pcnt):
        self.H, self.device = pages.shape[1], pages.device
        self.pages, self.pool, self.pcnt = pages, pool, pcnt
        self._wo = self._wml = None                        # split partials: grown, never freed (a captured graph may write
        self._retired = []                                 # into the ones it was given)

    def append(self, K, V, slots, reuse=False):
        """K, V [N, H, 128] bf16 (heads contiguous), slots int64 [N] = block * 16 + row, -1 = padding token"""
        kv_ext().append(K, V, slots, self.pages, self.pool, self.pcnt, reuse)

    def attention(self, q, block_table, lens, scale, splits=1, starts=None, min_pages=1, out=None):
        """one query token per sequence: q [B, Hq, 128] bf16 -> [B, Hq, 128] bf16"""
        B, Hq, _ = q.shape
        if out is None:
            out = torch.empty(B, Hq, 128, dtype=torch.bfloat16, device=q.device)
        if splits > 1:
            need = B * Hq * splits
            if self._wo is None or self._wo.numel() < need * 128:
                if self._wo is not None:
                    self._retired.append((self._wo, self._wml))
                self._wo = torch.empty(need * 128, dtype=torch.float32, device=q.device)
                self._wml = torch.empty(need * 2, dtype=torch.float32, device=q.device)
        else:
            if self._wo is None:
                self._wo = torch.empty(1, dtype=torch.float32, device=q.device)
                self._wml = torch.empty(1, dtype=torch.float32, device=q.device)
        kv_ext().attn(q, self.pages, self.pool, block_table, lens, out, self._wo, self._wml, scale, splits, starts,
                      min_pages)
        return out

    def chunk_attention(self, q, cu, block_table, lens, scale, splits=None, starts=None, out=None, window=0):
        """causal attention of several query tokens per sequence, after their keys and values have been appended: q [T, Hq, 128] bf16,
        sequence b's rows are cu[b] .. cu[b + 1] - 1 (cu int32 [B + 1]; None: one each), the last of them at position lens[b] - 1 ->
        [T, Hq, 128].  A query at position p sees tokens [max(starts, p - window + 1), p] (window 0: from starts on), one that sees none
        gives zeros; rows behind cu[B] of a given `out`, which lies apart from q, stay as they are.  splits: how many CTAs share a unit of rows
        (None: by the sizes, with the table's width for the context: a table no wider than the longest sequence splits best).  Values that
        are no numbers reach the queries that see them and no others (an infinity as itself, whatever it weighs).  Probabilities are rounded
        to BF16 for the product with the values, 2^-8 of each at most, as the output (attention() keeps some sixteen bits of them).  No gradients"""
        whole = 0
        if splits is None:
            splits, whole = chunk_splits(q.shape[0], block_table.shape[0], self.H, q.shape[1] // self.H, block_table.shape[1])
        host = calls()
        if host is not None:
            done = host[0].kv_chunk_attention(host[1], self.pages, self.pool, q, cu, block_table, lens, scale, splits, whole, starts, out,
                                              window)
            if done is not None:
                return done
        q = _rows(q, 128)
        if out is None:
            out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        need = lib().st_kv_chunk_attn_workspace_bytes(q.shape[0], q.shape[1], splits) // 4
        flat = torch.empty(need, dtype=torch.float32, device=q.device) if need else None
        wo, wml = (flat[:need // 130 * 128], flat[need // 130 * 128:]) if need else (None, None)
        kv_ext().chunk_attn(q, cu, self.pages, self.pool, block_table, lens, out, scale, splits, wo, wml, starts, window, whole)
        return out

    def dense(self, blocks=None):
        """pages (all, or the listed block ids) as exact BF16 Kd, Vd [n, 16, H, 128]"""
        n = self.pages.shape[0] if blocks is None else blocks.numel()
        Kd = torch.empty(n, PAGE, self.H, 128, dtype=torch.bfloat16, device=self.device)
        Vd = torch.empty_like(Kd)
        if blocks is None:
            kv_ext().dequant(self.pages, self.pool, Kd, Vd)
        else:
            kv_ext().dequant_blocks(self.pages, self.pool, blocks.to(torch.int32).contiguous(), Kd, Vd)
        return Kd, Vd

    def check(self):
        """raise if an escape could not be stored (extension pool exhausted): never silently lossy"""
        if int(self.pcnt[1].item()):
            raise RuntimeError("PagedKVCache: escape pool exhausted (pool_blocks too small)")

    def pool_usage(self):
        return int(self.pcnt[0].item()), self.pool.shape[0]

    def reset(self):
        self.pcnt.zero_()


def _rows(t, D):
    """t as the 8-bit kernels read it: heads contiguous, 16-byte aligned, token stride a multiple of 8 (copied if it is not)"""
    if t.numel() == 0 or (t.stride(2) == 1 and (t.stride(1) == D or t.size(1) == 1) and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def decode_splits8(units, max_pages, sms=148):
    """How many CTAs share a unit (sequence, KV head, eight query heads) of the 8-bit decode attention, from what the host knows: the
    number of units and the width of the block table.  Up to eight join on chip, as a cluster, which is a launch less; they are a power
    of two, since other clusters leave SMs idle (64 units of 1000 tokens: two 7.0 us, three 8.3, four 7.6; 256 of 4000: three 56.3,
    two 48.4).  Few units: eight up to 4096 tokens (8 units of 2000 tokens: 6.0 us, fifteen 7.0), one CTA of eight warps per SM beyond
    (8 units of 16000: eighteen 11.0, eight 14.2).  More: CTAs of four warps, four to an SM, so that sequences of different lengths
    even out (64 units of up to 16K tokens, lengths spread: two 43.6, eight 32.6; all of the full length 43.7 and 48.1).  Below 6, 8,
    16 or 64 pages per split the join costs more than it gives (128 units of 500 tokens: one 6.0, two 7.6)."""
    if units <= sms // 8:
        want, least = (8, 6) if max_pages <= 256 else (sms // max(1, units), 8)
    elif units <= 128:
        want, least = min(8, 4 * sms // units), 8 if units < 32 else 16
    else:
        want, least = 4 if units <= 4 * sms else 2, 64
    n = max(1, min(want, max_pages // least, 64))
    return n if n > 8 else 1 << n.bit_length() - 1


FEW_ROWS8 = 32      # rows (query, head of the group) per sequence up to which a chunk goes through the decode kernel (st_kv8_chunk.cu)


def chunk_splits8(tokens, seqs, kv_heads, group, max_pages, sms=148):
    """The same for a chunk of `tokens` queries of `seqs` sequences: a chunk of few rows per sequence is eight rows a CTA of the decode
    kernel, else 256 rows take an SM: split while that leaves SMs idle, down to 256 keys (one sequence of 4000 tokens, 64 rows, 8 KV
    heads: seven splits 21.6 us, sixteen 17.9)."""
    rows = -(-tokens * group // seqs)                       # of a sequence, on the mean
    if rows <= FEW_ROWS8:
        return decode_splits8(kv_heads * seqs * -(-rows // 8), max_pages, sms)
    return max(1, min(sms // (kv_heads * seqs * -(-rows // 256)), max_pages // 16, 64))


def chunk_splits(tokens, seqs, kv_heads, group, max_pages, sms=148):
    """(splits, whole) of the chunk attention over lossless pages, from what the host knows: how many CTAs share a unit of it, and how many
    units, the first ones, are not split.  A CTA takes an SM: 32 rows of a KV head for sequences of at most as many on the mean, else 256
    (st_kv_chunk.cu).  A step of 128 keys takes some 2 us, a CTA 10 besides; a join takes a launch, and every row's partial results go through
    memory.  Fewer units than SMs: split while that leaves SMs idle, down to 256 keys (512 queries behind 4000 tokens 95 us, in two 66;
    behind none 21 and 27).  A last wave that is part-filled, behind a long context: the full waves whole, the rest in as many splits as
    finish soonest (2048 queries behind 30000 tokens, 256 units on 148 SMs)."""
    seqs = max(1, seqs)
    rows = -(-tokens * group // seqs)                       # of a sequence, on the mean
    tile = 32 if rows <= 32 else 256
    units, steps = kv_heads * seqs * -(-rows // tile), (16 * max_pages - tokens // (2 * seqs)) / 128
    if units < 1:
        return 1, 0
    n = min(sms // units, max_pages // 16, 64)
    if n >= 2:
        return (n, 0) if 2.0 * steps * (1 - 1 / n) > 5 + 3e-4 * tokens * group * kv_heads * n else (1, 0)
    rest, before = units % sms, (16 * max_pages - tokens // seqs) / 128
    if rest == 0 or units > 4 * sms or before < 32:
        return 1, 0
    best, saved = 1, 0.0
    for n in (2, 3, 4, 5):
        gain = (1 - -(-rest * n // sms) / n) * 2.0 * before - (-(-rest * n // sms) - 1) * 10 - 5 - 3e-4 * min(tokens * group * kv_heads, rest * tile) * n
        if gain > saved:
            best, saved = n, gain
    if best == 1:
        return 1, 0
    empty = tokens * group // tile + seqs - units // kv_heads if seqs == 1 else 0      # (slots without rows come first)
    return best, units - rest + empty * kv_heads


class PageStore8:
    """Pages of one attention layer in 8 bits (256 B per token and head of dimension 128; a PageStore's take 400 and are lossless):
    pages uint8 [blocks, H, 2 (keys, values), 16, D] of e4m3 codes and exps int8 [blocks, H, 2], a value being e4m3(code) * 2^exp
    with one exponent per page, head and keys / values; the head dimension D is 64 or 128.  Same calls as PageStore; besides, append()
    takes a rotation and norms, and chunk_attention() several query tokens per sequence.  All calls go to the current stream, allocate
    only outputs and workspaces of their own (calls on several streams, and captured ones, do not meet there) and can be captured."""

    def __init__(self, num_blocks, num_kv_heads, device, head_dim=128):
        pages = torch.zeros(num_blocks, num_kv_heads, 2, PAGE, head_dim, dtype=torch.uint8, device=device)
        self._take(pages, torch.full((num_blocks, num_kv_heads, 2), -64, dtype=torch.int8, device=device))

    @classmethod
    def over(cls, pages, exps):
        """a store over page tensors that exist already (another store's, or part of a larger buffer), which are zero or written by
        append: the codes 0x7F and 0xFF, which it never writes, are no numbers and must not stand in a page that is read, masked rows
        included"""
        self = cls.__new__(cls)
        self._take(pages, exps)
        return self

    def _take(self, pages, exps):
        kv_ext()._pages8("PageStore8", pages, exps)
        self.pages, self.exps, self.device = pages, exps, pages.device
        self.H, self.D = pages.shape[1], pages.shape[4]
        self.marks = torch.zeros(17 * pages.shape[0], dtype=torch.int32, device=pages.device)    # the append's; zero between calls
        self.bad = torch.zeros(1, dtype=torch.int32, device=pages.device)

    def append(self, K, V, slots, positions=None, cos=None, sin=None, interleaved=True, q=None, q_norm=None, k_norm=None, eps=1e-6,
               q_out=None):
        """K, V [N, H, D] bf16, slots int64 [N] = block * 16 + row, -1 = padding token; the same slot twice: the last token counts.
        With cos / sin (float32 [P, D / 2]) keys are rotated at positions int64 [N] (or [1]: one for all), on pairs (2i, 2i + 1), or
        (i, i + D/2) with interleaved=False; with k_norm (bf16 [D]) they are RMS-normalised before.  q [N, Hq, D] goes the same way
        (q_norm) into q_out, which is returned.  A page is written from row 0 on: doing that again starts it anew (its other rows
        become zero); tokens that follow raise its exponent where they need to.  Appends that run at the same time (on two streams)
        must go to different pages."""
        host = calls()                                     # one native call for inputs that need no copy
        if host is not None:
            done = host[0].kv8_append(host[1], self.pages, self.exps, self.marks, self.bad, K, V, slots, positions, cos, sin, interleaved, q,
                                      q_norm, k_norm, eps, q_out)
            if done is not None:
                return done if q is not None else None
        K, V = _rows(K, self.D), _rows(V, self.D)
        if q is not None:
            q = _rows(q, self.D)
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        kv_ext().kv8_append(K, V, slots, self.pages, self.exps, self.marks, self.bad, positions, cos, sin, interleaved, k_norm, q, q_norm,
                            q_out, eps)
        return q_out

    def attention(self, q, block_table, lens, scale, splits=None, starts=None, min_pages=4, out=None, window=0):
        """one query token per sequence: q [B, Hq, D] bf16 -> [B, Hq, D] bf16; tokens [max(starts, lens - window), lens) take part
        (window 0: from starts on).  splits: how many CTAs share a sequence (None: by batch size and table width)"""
        if q.dim() == 3 and q.shape[1] > FEW_ROWS8 * self.H:    # (many heads to a KV head: rows enough for a tile)
            return self.chunk_attention(q, None, block_table, lens, scale, splits, starts, out, window)
        if splits is None:
            splits = decode_splits8(block_table.shape[0] * self.H * -(-q.shape[1] // (8 * self.H)), block_table.shape[1])
        host = calls()
        if host is not None:
            done = host[0].kv8_attention(host[1], False, self.pages, self.exps, q, None, block_table, lens, scale, splits, starts, min_pages,
                                         out, window)
            if done is not None:
                return done
        q = _rows(q, self.D)
        if out is None:
            out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        wo, wml = self._partials(q, block_table, splits, 0)
        kv_ext().kv8_attn(q, self.pages, self.exps, block_table, lens, out, scale, splits, wo, wml, starts, min_pages, window)
        return out

    def chunk_attention(self, q, cu, block_table, lens, scale, splits=None, starts=None, out=None, window=0):
        """causal attention of several query tokens per sequence, after their keys and values have been appended: q [T, Hq, D] bf16,
        sequence b's rows are cu[b] .. cu[b + 1] - 1 (cu int32 [B + 1]), the last of them at position lens[b] - 1 -> [T, Hq, D];
        rows behind cu[B] of a given `out` stay as they are"""
        if splits is None:
            seqs, group = max(1, block_table.shape[0]), max(1, q.shape[1] // self.H)
            splits = chunk_splits8(q.shape[0], seqs, self.H, group, block_table.shape[1])
        host = calls()
        if host is not None:
            done = host[0].kv8_attention(host[1], True, self.pages, self.exps, q, cu, block_table, lens, scale, splits, starts, 1, out, window)
            if done is not None:
                return done
        q = _rows(q, self.D)
        if out is None:
            out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        wo, wml = self._partials(q, block_table, splits, 1)
        kv_ext().kv8_chunk_attn(q, cu, self.pages, self.exps, block_table, lens, out, scale, splits, wo, wml, starts, window)
        return out

    def _partials(self, q, block_table, splits, chunk):
        """(wo, wml) of a call whose splits do not join on chip: its own, from the caching allocator"""
        need = lib().st_kv8_attn_workspace_bytes(q.shape[0], block_table.shape[0], q.shape[1], self.H, self.D, splits, chunk)
        if not need:
            return None, None
        flat = torch.empty(need // 4, dtype=torch.float32, device=q.device)
        rows = flat.numel() // (self.D + 2)
        return flat[:rows * self.D], flat[rows * self.D:]

    def dense(self, blocks=None):
        """pages (all, or the listed block ids) as exact BF16 Kd, Vd [n, 16, H, D]"""
        host = calls()
        if host is not None:
            done = host[0].kv8_dense(host[1], self.pages, self.exps, blocks)
            if done is not None:
                return done
        n = self.pages.shape[0] if blocks is None else blocks.numel()
        Kd = torch.empty(n, PAGE, self.H, self.D, dtype=torch.bfloat16, device=self.device)
        Vd = torch.empty_like(Kd)
        kv_ext().kv8_dequant_blocks(self.pages, self.exps, None if blocks is None else blocks.to(torch.int32).contiguous(), Kd, Vd)
        return Kd, Vd

    def check(self):
        """raise if a value that is not finite (or beyond 448 * 2^56) was appended: it was cut off, a NaN stored as zero"""
        if int(self.bad.item()):
            raise RuntimeError("PageStore8: values that are not finite were appended")

    def reset(self):
        self.bad.zero_()


class PagedKVCache:
    """Static paged cache for a decoder: per-layer pages, one block table [B, max_pages] (sequence b owns pages
    b * max_pages ...), a GPU-side token count so decode steps are CUDA-graph safe.  eight_bit: the layers are PageStore8s (heads of
    head_dim 64 or 128), which take 256 B per token and head of 128 for the 400 of the lossless pages."""

    def __init__(self, num_layers, batch_size, max_cache_len, num_kv_heads, device, pool_blocks=1 << 15, eight_bit=False, head_dim=128):
        self.B = batch_size
        self.max_pages = (max_cache_len + PAGE - 1) // PAGE
        self.max_len = self.max_pages * PAGE
        self.device = torch.device(device)
        self.eight_bit = eight_bit
        blocks = batch_size * self.max_pages
        self.layers = [PageStore8(blocks, num_kv_heads, device, head_dim) if eight_bit else PageStore(blocks, num_kv_heads, device, pool_blocks)
                       for _ in range(num_layers)]
        self.bt32 = torch.arange(batch_size * self.max_pages, dtype=torch.int32, device=device).view(batch_size, -1)
        self.bt64 = self.bt32.long()
        self.lens = torch.zeros(batch_size, dtype=torch.int32, device=device)
        self.cum = torch.zeros((), dtype=torch.long, device=device)      # tokens stored (same for every sequence)
        self._stored = 0                                                  # the same count on the host, for capacity checks

    def update(self, layer_idx, key_states, value_states):
        """key/value_states [B, H, T, 128]; positions continue from the GPU-side count; returns the slots used"""
        B, H, T, D = key_states.shape
        self._stored += T if layer_idx == len(self.layers) - 1 else 0
        if self._stored + (T if layer_idx != len(self.layers) - 1 else 0) > self.max_len:
            raise ValueError(f"PagedKVCache.update: position {self._stored + T} exceeds the capacity of "
                             f"{self.max_len} tokens")
        slots = self.next_slots(B, T)
        K = key_states.transpose(1, 2).reshape(B * T, H, D)
        V = value_states.transpose(1, 2).reshape(B * T, H, D)
        self.layers[layer_idx].append(K.contiguous(), V.contiguous(), slots)
        if layer_idx == len(self.layers) - 1:
            self.cum += T
            self.lens[:B] = self.cum.to(torch.int32)
        elif layer_idx == 0:
            self.lens[:B] = (self.cum + T).to(torch.int32)
        return slots

    def next_slots(self, B, T):
        """slots [B * T] of the next T tokens of every sequence (sequence after sequence)"""
        cp = torch.arange(T, device=self.device) + self.cum
        return (self.bt64[:B][:, cp // PAGE] * PAGE + (cp % PAGE)).reshape(-1)

    def begin_chunk(self, B, T):
        """the next T tokens of every sequence, for all layers: their slots; lens counts them.  end_chunk(T) closes the chunk"""
        if self._stored + T > self.max_len:
            raise ValueError(f"PagedKVCache.begin_chunk: position {self._stored + T} exceeds the capacity of {self.max_len} tokens")
        slots = self.next_slots(B, T)
        self.lens[:B] = (self.cum + T).to(torch.int32)
        return slots

    def end_chunk(self, T):
        self._stored += T
        self.cum += T

    def begin_step(self, B):
        """decode step (one token per sequence): the slots every layer appends at, computed once; lens counts the new
        token.  Graph-safe (positions come from the GPU-side count)."""
        if self.cum.is_cuda and B <= self.B:
            slots = torch.empty(B, dtype=torch.long, device=self.cum.device)
            kv_ext().decode_slots(self.cum, self.bt64[:B], self.max_len, slots, self.lens)
            return slots
        page = (self.cum // PAGE).clamp(max=self.max_pages - 1)            # a full cache never indexes past the table:
        slots = self.bt64[:B].gather(1, page.expand(B, 1)).view(B) * PAGE + self.cum % PAGE
        slots = torch.where(self.cum < self.max_len, slots, torch.full_like(slots, -1))   # ... the token is dropped
        self.lens[:B] = (self.cum + 1).clamp(max=self.max_len).to(torch.int32)
        return slots

    def end_step(self):
        self.cum += 1

    def attention(self, layer_idx, q, scale, splits=None):
        """decode step: q [B, Hq, 128] against everything stored in the layer (including this step's token)"""
        B = q.shape[0]
        if splits is None and not self.eight_bit:
            splits = decode_splits(B, self.layers[layer_idx].H, self.max_pages)
        return self.layers[layer_idx].attention(q, self.bt32[:B], self.lens[:B], scale, splits, None, 4)

    def check(self):
        for layer in self.layers:
            layer.check()

    def reset(self):
        self._stored = 0
        self.cum.zero_()
        self.lens.zero_()
        for layer in self.layers:
            layer.reset()


try:                                                   # the transformers glue, under the reference's names
    from .hf_cache import StateTreeKVCache, StateTreeKVLayer, enable, statetree_attention  # noqa: E402,F401
except ImportError:                                    # transformers absent or too old: the page store still works
    pass
