"""Paged KV cache: sequences of their own lengths over one pool of fixed-size pages.

``OPDStaticCache`` keeps one shared length (shorter sequences are left-padded and every row
holds the longest one's capacity), which is what the verify loop of the reference expects. For
plain decoding of ragged batches this module keeps pages instead: a sequence holds the pages its
own length needs, sequences are admitted and released by handing pages out and back, and nothing
moves. The reference has no such cache.

``paged_append`` stores new K/V rows, rotating K (and the queries, in the same launch) by their
positions on the way; ``paged_attention`` is the attention of one new token per sequence;
``PagedKVCache`` keeps the pages, tables and lengths, and is a transformers ``Cache`` for models
whose attention is this package's ('speckv_tree').
"""
import torch
from transformers.cache_utils import Cache

from . import _ops


def paged_append(key, value, key_pages, value_pages, page_table, starts, *, counts=None, query=None, rotation=None,
                 positions=None, interleaved=False, query_out=None):
    """Stores row t of sequence b at position starts[b] + t of a paged cache and returns the
    rotated queries (None without ``query``), in one launch.

    ``key`` / ``value`` (batch, kv_heads, rows, head_dim) strided views; ``key_pages`` /
    ``value_pages`` (pages, kv_heads, page_size, head_dim) of the same dtype (bf16 / fp16 / fp32);
    ``page_table`` (batch, pages) int64 names the pool page of each page_size positions;
    ``starts`` (batch,) int64. ``counts`` (batch,) int64: rows t >= counts[b] are padding, not
    read or stored (None: all rows are live).
    ``rotation = (cos, sin)``, float32 (positions, rotation_dim / 2) tables, turns the first
    rotation_dim dims of ``key`` and ``query`` (batch, q_heads, rows, head_dim), in halves or,
    ``interleaved``, in neighbouring pairs, by row ``positions[b, t]`` (int64; None: the cache
    position). Queries of padding rows come back as zeros. ``query_out`` may be ``query`` itself.
    A page outside the pools, a position the table or the rotation does not hold: that token is
    treated as padding and reported by ``_ops.device_error``. No two live tokens of a call may
    name the same slot. Inference only: no gradient flows through it.
    """
    return _ops.paged_append(key, value, key_pages, value_pages, page_table, starts, counts, query, rotation,
                             positions, interleaved, query_out)


def paged_attention(query, key_pages, value_pages, page_table, lengths, scale=None, *, out=None):
    """softmax(scale q k) v of one new token per sequence over its first lengths[b] positions.

    ``query`` (batch, q_heads, 1, head_dim); pools and ``page_table`` as for ``paged_append``;
    ``lengths`` (batch,) int64. Query head h reads KV head h // (q_heads // kv_heads). A sequence
    of length 0 gives zeros, an infinite value makes its outputs infinite or NaN. fp32 products are
    taken to 2^-21 and summed in fp32 (a value within 2^-12 of the type's largest counts as
    infinite). Returns (batch, 1, q_heads, head_dim). Head dims to 256. Inference only: no gradient
    flows through it.
    """
    return _ops.paged_attention(query, key_pages, value_pages, page_table, lengths,
                                query.shape[-1] ** -0.5 if scale is None else scale, out)


def rotation_tables(positions, rotation_dim, theta=10000.0, device='cuda'):
    """(cos, sin) float32 tables of paged_append, of angles computed in 64 bits."""
    if rotation_dim < 2 or rotation_dim % 2 or positions < 1:
        raise ValueError('rotation_tables: an even rotation_dim and at least one position required')
    freq = float(theta) ** (-torch.arange(0, rotation_dim, 2, device=device, dtype=torch.float64) / rotation_dim)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


class PagedKVCache(Cache):
    """Pools, page tables and lengths of a batch of sequences; one table for all layers.

    A forward over new tokens is ``begin(counts)`` (pages for them, positions fixed), then per
    layer ``append`` and ``attend``. ``admit`` adds empty sequences at the end of the batch,
    ``release`` drops finished ones (the last sequences take their places, as
    ``swap_remove_plan`` has it) and hands their pages back. Sizes live on the host; the table
    and lengths are copied to the device on the current stream, into the same memory each time: the
    ``append`` and ``attend`` calls of a step may be captured into a CUDA graph (every layer's pools made
    before), and replayed after each ``begin`` over as many tokens of as many sequences from the same
    first one. ``begin`` and ``release`` stay outside the capture.

    As a transformers cache: ``update`` begins a forward at layer 0. Prompts go through empty
    sequences, right-padded (``prompt_lengths`` says how long each is); afterwards one token per
    sequence at a time. The model's attention must be this package's, and position ids are the
    caller's: ``lengths`` before the forward.
    """

    def __init__(self, pages, page_size=64, *, batch_capacity, max_length):
        if pages < 1 or page_size < 1 or batch_capacity < 1 or max_length < 1:
            raise ValueError('positive pages, page_size, batch_capacity and max_length required')
        try:
            super().__init__(layers=[])
        except TypeError:
            super().__init__()
            self.layers = []
        self.page_size, self.batch_capacity, self.max_length = page_size, batch_capacity, max_length
        self.table_pages = -(-max_length // page_size)
        self.pages = pages
        self.lengths = []            # of each live sequence, rows of a begun forward included
        self._held = []              # pool pages of each live sequence, in order
        self._free = list(range(pages - 1, -1, -1))
        self._pools = []             # (key_pages, value_pages) per layer, created on first use
        self._table = None           # (batch_capacity, table_pages) int64 on the device
        self._numbers = None         # (3 * batch_capacity,) int64 there: starts, counts, lengths of the begun forward
        self._device = None
        self._step = None            # (first, starts, counts, lengths) device views of it
        self._rows = 0               # the most new tokens of a sequence in it
        self._prompts, self._prompt_mask = None, {}

    # ---- sequences -----------------------------------------------------------
    @property
    def free_pages(self):
        return len(self._free)

    def page_table(self, first=0, count=None):
        count = len(self.lengths) - first if count is None else count
        return self._table[first:first + count]

    def admit(self, count):
        """Adds `count` empty sequences at the end of the batch; returns their first index."""
        first = len(self.lengths)
        if count < 0 or first + count > self.batch_capacity:
            raise ValueError(f'{count} more sequences exceed the batch capacity of {self.batch_capacity}')
        self.lengths += [0] * count
        self._held += [[] for _ in range(count)]
        return first

    def release(self, finished):
        """Drops the sequences whose entry of `finished` (one per live sequence) is true. Returns
        the old index of each remaining sequence (holes are filled from the batch's end)."""
        from .opd_static_cache import swap_remove_plan
        if len(finished) != len(self.lengths):
            raise ValueError('one entry per live sequence required')
        self._outside_capture('release')
        for i, done in enumerate(finished):
            if done:
                self._free += reversed(self._held[i])
        keep, _, _ = swap_remove_plan(finished)
        self.lengths = [self.lengths[i] for i in keep]
        self._held = [self._held[i] for i in keep]
        self._step = None
        if self._table is not None and keep:
            self._upload_table(range(len(keep)))
        return keep

    def _upload_table(self, rows):
        rows = list(rows)
        staged = torch.zeros((len(rows), self.table_pages), dtype=torch.long)
        for i, r in enumerate(rows):
            if self._held[r]:
                staged[i, :len(self._held[r])] = torch.tensor(self._held[r], dtype=torch.long)
        if rows == list(range(rows[0], rows[0] + len(rows))):
            self._table[rows[0]:rows[0] + len(rows)].copy_(self._pin(staged), non_blocking=True)
        else:
            self._table[torch.tensor(rows, device=self._device)] = staged.to(self._device)

    def _outside_capture(self, what):
        if self._device is not None and self._device.type == 'cuda' and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f'{what}() decides and copies on the host: call it before a captured graph is replayed, '
                               'not inside its capture')

    def _pin(self, t):
        return t.pin_memory() if self._device.type == 'cuda' else t

    # ---- a forward over new tokens ---------------------------------------------
    def begin(self, counts=1, first=0, *, device=None):
        """Starts a forward over counts[i] new tokens (an int: the same for all) of sequence
        first + i: hands out the pages they need and fixes their positions."""
        self._step = None  # a begin that raises leaves no forward behind
        live = len(self.lengths)
        if isinstance(counts, int):
            counts = [counts] * (live - first)
        counts = [int(c) for c in counts]
        if first < 0 or first + len(counts) > live or any(c < 0 for c in counts):
            raise ValueError('token counts of live sequences required')
        ends = [self.lengths[first + i] + c for i, c in enumerate(counts)]
        if ends and max(ends) > self.max_length:
            raise ValueError(f'a sequence of {max(ends)} positions exceeds max_length {self.max_length}')
        wants = [max(0, -(-e // self.page_size) - len(self._held[first + i])) for i, e in enumerate(ends)]
        if sum(wants) > len(self._free):
            raise RuntimeError(f'{sum(wants)} pages needed, {len(self._free)} free')
        if self._device is None:
            self._device = torch.device(device if device is not None else 'cuda')
        self._outside_capture('begin')
        if self._table is None:
            with torch.inference_mode(False):  # written again in either mode
                self._table = torch.zeros((self.batch_capacity, self.table_pages), dtype=torch.long, device=self._device)
                self._numbers = torch.zeros(3 * self.batch_capacity, dtype=torch.long, device=self._device)
            self._device = self._table.device
        for i, want in enumerate(wants):
            for _ in range(want):
                self._held[first + i].append(self._free.pop())
        grown = [first + i for i, want in enumerate(wants) if want]
        if grown:
            self._upload_table(grown)
        staged = torch.tensor([self.lengths[first:first + len(counts)], counts, ends], dtype=torch.long)
        numbers = self._numbers[:staged.numel()].view(staged.shape)
        numbers.copy_(self._pin(staged), non_blocking=True)
        starts, counts_dev, lengths = numbers.unbind(0)
        self.lengths[first:first + len(counts)] = ends
        self._step, self._rows = (first, starts, counts_dev, lengths), max(counts, default=0)

    def _layer_pools(self, layer, key):
        while len(self._pools) <= layer:
            self._pools.append(None)
        if self._pools[layer] is None:
            shape = (self.pages, key.shape[1], self.page_size, key.shape[3])
            self._pools[layer] = (torch.empty(shape, dtype=key.dtype, device=key.device),
                                  torch.empty(shape, dtype=key.dtype, device=key.device))
        return self._pools[layer]

    def _begun(self, batch):
        if self._step is None or self._step[1].numel() != batch:
            raise RuntimeError('begin() a forward over these sequences first')
        return self._step

    def append(self, key, value, layer, *, query=None, rotation=None, positions=None, interleaved=False):
        """Stores the begun forward's K/V rows of `layer`; returns the rotated queries."""
        first, starts, counts, _ = self._begun(key.shape[0])
        if key.shape[2] < self._rows:
            raise ValueError(f'{key.shape[2]} rows for a forward begun over up to {self._rows} new tokens')
        k_pages, v_pages = self._layer_pools(layer, key)
        return _ops.paged_append(key, value, k_pages, v_pages, self.page_table(first, key.shape[0]), starts, counts,
                                 query, rotation, positions, interleaved)

    def attend(self, query, layer, scale=None):
        """Attention of one new token per sequence over `layer`, the begun forward's rows included."""
        first, _, _, lengths = self._begun(query.shape[0])
        k_pages, v_pages = self._pools[layer]
        return paged_attention(query, k_pages, v_pages, self.page_table(first, query.shape[0]), lengths, scale)

    # ---- transformers cache ------------------------------------------------------
    def prompt_lengths(self, lengths):
        """Lengths of the right-padded prompts of the next forward (None: every row is live). They hold for
        that forward alone, whether it succeeds or not; ``reset`` drops them too."""
        self._prompts = None if lengths is None else [int(n) for n in lengths]

    def _begin_update(self, batch, rows, device):
        prompts, self._prompts, self._prompt_mask = self._prompts, None, {}
        fresh = not self.lengths
        if fresh:
            self.admit(batch)
        try:
            if batch != len(self.lengths):
                raise ValueError('KV batch differs from live request count')
            if rows > 1 and any(self.lengths):
                raise ValueError('after its prompt a paged cache takes one token per sequence at a time')
            counts = prompts if prompts is not None else [rows] * batch
            if len(counts) != batch or any(not 0 <= c <= rows for c in counts):
                raise ValueError('prompt lengths do not match the prompt rows')
            self.begin(counts, device=device)
        except Exception:
            if fresh:  # the sequences of a prompt that did not enter
                self._drop_all()
            raise

    def update(self, key_states, value_states, layer_idx, *args, **kwargs):
        batch, rows = key_states.shape[0], key_states.shape[2]
        if layer_idx == 0:
            self._begin_update(batch, rows, key_states.device)
        self.append(key_states, value_states, layer_idx)
        if rows > 1:  # the prompt attends to itself: its own rows are all there is
            key_states._speckv_prompt = self._prompt_mask
            return key_states, value_states
        first, _, _, lengths = self._step
        k_pages, v_pages = (pool[:] for pool in self._pools[layer_idx])
        k_pages._speckv_pages = v_pages._speckv_pages = (self.page_table(first, batch), lengths)
        return k_pages, v_pages

    def get_seq_length(self, layer_idx=0):
        return max(self.lengths, default=0)

    def get_mask_sizes(self, query_length, layer_idx=0):
        return self.get_seq_length() + (query_length if isinstance(query_length, int) else len(query_length)), 0

    def get_max_cache_shape(self, layer_idx=0):
        return self.max_length

    def __len__(self):
        return len(self._pools)

    def __bool__(self):
        return bool(self.lengths)

    def reset(self):
        """Drops every sequence and the next forward's prompt lengths; the pools stay."""
        self._prompts = None
        self._drop_all()

    def _drop_all(self):
        for held in self._held:
            self._free += reversed(held)
        self.lengths, self._held, self._step = [], [], None

    def _unsupported(self, *args, **kwargs):
        raise NotImplementedError('a paged cache admits and releases whole sequences (admit, release); its rows are '
                                  'not cropped, reordered or repeated')

    crop = reorder_cache = batch_repeat_interleave = batch_select_indices = _unsupported

    def statistics(self):
        return {'pages': self.pages, 'free_pages': len(self._free), 'sequences': len(self.lengths),
                'kv_cache_bytes': sum(p.numel() * p.element_size() for pair in self._pools if pair for p in pair)}
