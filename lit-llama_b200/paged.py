"""Paged key/value caches: the keys and values of many sequences in the pages of one pool, for serving sequences whose lengths are not known beforehand.

    PagePool     which sequence has which pages (host side): sequences come, grow and go, a step books what it needs
    PagedStep    one step's sequences on the device: rows, lengths, page tables.  Made once, used by every layer
    PagedCache   one layer's pool: `write` (quantising e4m3 or int8 pools as rows come), `read`, and `attend`, causal softmax attention of the step's new
                 tokens, single ones and chunks together, over all that the pool holds of their sequences; with a window the last `window`
                 positions and the first `first` ones

        pool = PagePool(n_pages=4096, page=64, device="cuda")
        caches = [PagedCache.empty(4096, 64, kv_heads=8, dim=128, dtype=torch.bfloat16, store="fp8") for _ in layers]
        step = pool.step([("a", 512), ("b", 1)])               # 512 new tokens of a, one of b: rows 0..511 and 512
        caches[i].write(k, v, step)                            # k [513, 8, 128], v [513, 8, 128]
        out = caches[i].attend(q, step)                        # q [513, 32, 128] -> [513, 32, 128]
        pool.release("a")

A token's key and value rows are quantised by themselves, per head: scale = max(max |x| (1 / c), 2^-126), code = round(x / scale), c = 448 (fp8, e4m3) or 127
(int8).  A row that holds an infinity or NaN reads back as NaN.  A row whose weights sum to zero (it sees no key) attends to zeros.  Everything
is a kernel of libb200seq (include/b2l_seq.h); CUDA only, no CPU fallback, no derivatives."""
from typing import Dict, Hashable, List, Mapping, Optional, Sequence, Tuple

import torch

from . import _seqlib as S
from .state import PagesFull

STORES = {"act": S.STORE_ACT, "fp8": S.STORE_E4M3, "int8": S.STORE_INT8}
PAGES = (16, 32, 64, 128, 256)


class PagedStep:
    """One step's sequences: sequence b has rows starts[b] .. starts[b + 1] - 1 of the step's tokens, is lengths[b] tokens long with them, and its token j
    lies in page table[b, j // page].  An entry of the table outside the pool (-1) is a page that is not there: its keys are not seen.

    The tensors (int32, on the device) may be overwritten between replays of a graph that was recorded with them.  `rows` is the number of tokens;
    max_new and max_length are what the host knows of the sequences' most new tokens and lengths: they pick between equivalent forms (every form is right for
    every content of the tensors), so they should be about right."""

    def __init__(self, starts: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor, *, rows: int, max_new: int = 0, max_length: int = 0) -> None:
        for name, t, dims in (("starts", starts, 1), ("lengths", lengths, 1), ("table", table, 2)):
            if t.dtype != torch.int32 or t.dim() != dims or t.stride(-1) != 1:
                raise ValueError(f"paged step: {name} must be int32 with {dims} dimension(s), its entries consecutive")
            if t.device != lengths.device:
                raise ValueError("paged step: its tensors are on different devices")
        if starts.numel() != lengths.numel() + 1 or table.shape[0] != lengths.numel() or table.shape[1] < 1:
            raise ValueError(f"paged step: {lengths.numel()} lengths, {starts.numel()} starts (one more is wanted), a table of {tuple(table.shape)}")
        if rows < 0:
            raise ValueError("paged step: a negative number of rows")
        self._tensors, self.rows, self.seqs = (starts, lengths, table), int(rows), lengths.numel()
        self.device = lengths.device
        self.max_new, self.max_length = max(int(max_new), 0), max(int(max_length), 0)
        self._at = (S.ptr(starts), S.ptr(lengths), S.ptr(table), table.stride(0), table.shape[1]) if lengths.is_cuda else None
        self._plans: Dict[tuple, tuple] = {}                                # of attend: what does not change from layer to layer

    # the kernels have the tensors' addresses: their contents may change, they stay
    starts = property(lambda self: self._tensors[0])
    lengths = property(lambda self: self._tensors[1])
    table = property(lambda self: self._tensors[2])

    @classmethod
    def of(cls, sequences: Sequence[Tuple[int, int, Sequence[int]]], device, *, width: int = 0) -> "PagedStep":
        """From the host: (new tokens, length with them, pages) of every sequence; `width`: the table's, at least the longest list of pages."""
        starts, lengths, rows = [0], [], 0
        width = max([int(width), 1] + [len(p) for _, _, p in sequences])
        flat: List[int] = []
        for new, length, pages in sequences:
            if new < 0 or length < new:
                raise ValueError(f"paged step: {new} new tokens of a sequence that is {length} long with them")
            rows += new
            starts.append(rows)
            lengths.append(length)
            flat += list(pages) + [-1] * (width - len(pages))
        n = len(lengths)
        both = torch.tensor(starts + lengths + flat, dtype=torch.int32).to(device)
        return cls(both[:n + 1], both[n + 1:2 * n + 1], both[2 * n + 1:].view(n, width), rows=rows,
                   max_new=max((new for new, _, _ in sequences), default=0), max_length=max(lengths, default=0))

    def refill(self, other: "PagedStep") -> None:
        """The other step's sequences in this one's tensors (of the same number of sequences and rows, and at least its width), for a graph that was
        recorded with this one."""
        if other.seqs != self.seqs or other.rows != self.rows or other.table.shape[1] > self.table.shape[1]:
            raise ValueError(f"paged step: {other.seqs} sequences with {other.rows} rows and {other.table.shape[1]} pages do not fit {self.seqs} with {self.rows} and {self.table.shape[1]}")
        self.starts.copy_(other.starts, non_blocking=True)
        self.lengths.copy_(other.lengths, non_blocking=True)
        self.table[:, :other.table.shape[1]].copy_(other.table, non_blocking=True)
        self.table[:, other.table.shape[1]:].fill_(-1)


class PagePool:
    """Which sequence has which of `n_pages` pages.  With a window, pages that neither the window nor the first `first` positions reach any more
    are given back as a sequence grows (their place in its table becomes -1): for models whose layers all look back no further."""

    def __init__(self, n_pages: int, page: int, device, *, window: int = 0, first: int = 0) -> None:
        if n_pages < 1 or page not in PAGES:
            raise ValueError(f"page pool: {n_pages} pages of {page} tokens: at least one, of {PAGES}")
        if window < 0 or first < 0:
            raise ValueError("page pool: a negative window or number of first tokens")
        self.n_pages, self.page, self.device, self.window, self.first = int(n_pages), int(page), torch.device(device), int(window), int(first)
        self._free: List[int] = list(range(self.n_pages - 1, -1, -1))       # page 0 first
        self._pages: Dict[Hashable, List[int]] = {}
        self._length: Dict[Hashable, int] = {}

    def has(self, request_id: Hashable) -> bool:
        return request_id in self._pages

    def requests(self) -> List[Hashable]:
        return list(self._pages)

    def free_pages(self) -> int:
        return len(self._free)

    def position(self, request_id: Hashable) -> int:
        """Tokens of the sequence so far."""
        return self._length[request_id]

    def pages(self, request_id: Hashable) -> List[int]:
        return list(self._pages[request_id])

    def most_pages(self, tokens: int, portion: int = 0) -> int:
        """The most pages at a time of a sequence that grows to `tokens` tokens, at most `portion` of them in a step (0: any number)."""
        whole = -(-tokens // self.page)
        if not self.window:
            return whole
        reach = self.window - 1 + (min(portion, tokens) if portion else tokens)      # positions that a step's tokens see or are
        return min(whole, -(-self.first // self.page) + (reach + 2 * self.page - 2) // self.page)

    def has_room(self, live: Mapping[Hashable, int], tokens: int, portion: int = 0) -> bool:
        """Whether one more sequence, of `tokens` tokens, finds its pages whatever the sequences of `live` (request id -> the tokens that it grows to) still
        take.  Other sequences are counted with the pages that they have."""
        held = sum(sum(p >= 0 for p in self._pages.get(rid, ())) for rid in live)
        return len(self._free) + held >= sum(self.most_pages(n, portion) for n in live.values()) + self.most_pages(tokens, portion)

    def release(self, request_id: Hashable) -> None:
        self._free += [p for p in reversed(self._pages.pop(request_id)) if p >= 0]
        del self._length[request_id]

    def take_back(self, request_id: Hashable, n: int) -> None:
        """The last n tokens that were booked for a sequence did not come: it is as long as it was, and pages of theirs alone are free again."""
        if not 0 <= n <= self._length[request_id]:
            raise ValueError(f"page pool: {n} tokens of {self._length[request_id]}")
        length = self._length[request_id] - n
        pages, keep, reach = self._pages[request_id], -(-length // self.page), length - self.window + 1
        if any(p < 0 and (i * self.page < self.first or (i + 1) * self.page > reach) for i, p in enumerate(pages[:keep])):
            raise ValueError(f"page pool: pages that the window at {length} reaches were given back")
        self._length[request_id] = length
        self._free += [p for p in reversed(pages[keep:]) if p >= 0]
        del pages[keep:]

    def _behind(self, request_id: Hashable) -> List[int]:
        """Places in the sequence's table that no later token sees."""
        if not self.window or request_id not in self._pages:
            return []
        reach = self._length[request_id] - self.window + 1                  # the first position that the next token's window has
        return [i for i, p in enumerate(self._pages[request_id]) if p >= 0 and i * self.page >= self.first and (i + 1) * self.page <= reach]

    def step(self, entries: Sequence[Tuple[Hashable, int]], *, width: int = 0) -> PagedStep:
        """Books `n` more tokens for every (request id, n); ids that are not known begin a sequence.  Raises PagesFull, with nothing booked, where the
        pages do not suffice."""
        if len({rid for rid, _ in entries}) < len(entries):
            raise ValueError("page pool: a request comes twice in one step")
        if any(n < 0 for _, n in entries):
            raise ValueError("page pool: a negative number of tokens")
        behind, new = {rid: self._behind(rid) for rid, _ in entries}, {rid for rid, _ in entries if rid not in self._pages}
        need = sum(max(0, -(-(self._length.get(rid, 0) + n) // self.page) - len(self._pages.get(rid, ()))) for rid, n in entries)
        if need > len(self._free) + sum(len(b) for b in behind.values()):
            raise PagesFull(f"{need} pages are needed, {len(self._free)} of {self.n_pages} are free")
        sequences = []
        for rid, _ in entries:
            for i in behind[rid]:
                self._free.append(self._pages[rid][i])
                self._pages[rid][i] = -1
        for rid, n in entries:
            pages = self._pages.setdefault(rid, [])
            self._length[rid] = self._length.get(rid, 0) + n
            while len(pages) * self.page < self._length[rid]:
                pages.append(self._free.pop())
            sequences.append((n, self._length[rid], pages))
        try:
            return PagedStep.of(sequences, self.device, width=width)
        except BaseException:                                               # no memory on the device
            for rid, n in entries:
                self.take_back(rid, n)
                if rid in new:
                    self.release(rid)
            raise


class PagedCache:
    """One layer's pool: keys [pages, kv_heads, page, dim] and values [pages, kv_heads, page, vdim] in the activation type (bf16 or f32), in e4m3
    (torch.float8_e4m3fn) or in int8, the 8-bit ones with f32 scales [pages, kv_heads, page].  `dtype`: the activation type of an 8-bit pool."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, *,
                 dtype: Optional[torch.dtype] = None) -> None:
        if k.dtype != v.dtype or k.dim() != 4 or v.dim() != 4 or k.shape[:3] != v.shape[:3] or k.device != v.device:
            raise ValueError(f"paged cache: keys {tuple(k.shape)} {k.dtype} and values {tuple(v.shape)} {v.dtype} do not belong together")
        if k.dtype in (torch.float8_e4m3fn, torch.int8):
            self.store, self.dtype = ("fp8" if k.dtype == torch.float8_e4m3fn else "int8"), dtype or torch.bfloat16
            for s in (k_scale, v_scale):
                if s is None or s.dtype != torch.float32 or s.shape != k.shape[:3] or s.device != k.device or not s.is_contiguous():
                    raise ValueError(f"paged cache: an 8-bit pool needs contiguous f32 scales {tuple(k.shape[:3])}")
        else:
            self.store, self.dtype = "act", dtype or k.dtype
            if k_scale is not None or v_scale is not None:
                raise ValueError("paged cache: scales belong to an 8-bit pool")
            if self.dtype != k.dtype:
                raise ValueError(f"paged cache: a pool in {k.dtype} for activations in {self.dtype}")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("paged cache: the pool must be contiguous")
        self._pool = (k, v, k_scale, v_scale)
        (self.n_pages, self.kv_heads, self.page, self.dim), self.vdim = k.shape, v.shape[3]
        if self.n_pages < 1 or self.kv_heads < 1 or self.page not in PAGES:
            raise ValueError(f"paged cache: {self.n_pages} pages of {self.kv_heads} heads, {self.page} tokens: at least one, of {PAGES}")
        if any(d < 16 or d > 256 or d % 16 for d in (self.dim, self.vdim)):
            raise ValueError(f"paged cache: heads of {self.dim} and {self.vdim} entries: multiples of 16 up to 256")
        self.device = k.device
        self._codes = (STORES[self.store], S.act_code(self.dtype))
        self._sizes = (self.n_pages, self.page, self.kv_heads, self.dim, self.vdim) + self._codes
        self._like = torch.empty(0, dtype=self.dtype, device=k.device)
        self._per = 4 if self.dtype == torch.float32 else 8                 # entries in 16 bytes
        self._at = tuple(S.ptr(t) for t in (k, v, k_scale, v_scale)) if k.is_cuda else None

    # the kernels have the tensors' addresses: their contents may change, they stay
    k = property(lambda self: self._pool[0])
    v = property(lambda self: self._pool[1])
    k_scale = property(lambda self: self._pool[2])
    v_scale = property(lambda self: self._pool[3])

    @classmethod
    def empty(cls, n_pages: int, page: int, kv_heads: int, dim: int, vdim: Optional[int] = None, *, dtype: torch.dtype = torch.bfloat16, store: str = "act",
              device="cuda") -> "PagedCache":
        """A pool of zeros."""
        if store not in STORES:
            raise ValueError(f"paged cache: store {store!r}: one of {sorted(STORES)}")
        kept = {"act": dtype, "fp8": torch.float8_e4m3fn, "int8": torch.int8}[store]
        shape = (int(n_pages), int(kv_heads), int(page))
        k, v = (torch.zeros(shape + (int(d),), dtype=kept, device=device) for d in (dim, vdim or dim))
        scales = [torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(2)] if store != "act" else [None, None]
        return cls(k, v, *scales, dtype=dtype)

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._pool if t is not None)

    # ------------------------------------------------------------------ calls (of every layer and step: some 5 us each beside the launches)
    def _rows(self, x: torch.Tensor, heads: int, size: int, step: PagedStep, what: str) -> Tuple[torch.Tensor, int, int]:
        """x [rows, heads, size] as the kernels take it, entries of a head consecutive and rows on 16-byte borders (else a copy), with the entries between its
        rows and between its heads."""
        shape = x.shape
        if len(shape) != 3 or shape[2] != size or (heads and shape[1] != heads) or x.dtype is not self.dtype or x.device != self.device:
            raise ValueError(f"paged cache: {what} {tuple(shape)} {x.dtype} on {x.device}, [rows, {heads or 'heads'}, {size}] {self.dtype} on {self.device} is wanted")
        if shape[0] < step.rows:
            raise ValueError(f"paged cache: {what} has {shape[0]} rows, the step {step.rows}")
        s0, s1, s2 = x.stride()
        if shape[1] == 1:                                                   # of one head or row: whatever torch says
            s1 = size
        if shape[0] == 1:
            s0 = shape[1] * size
        if s2 != 1 or s0 % self._per or s1 % self._per or x.data_ptr() % 16:
            x = x.contiguous()
            if x.data_ptr() % 16:
                x = x.clone(memory_format=torch.contiguous_format)
            s0, s1 = shape[1] * size, size
        return x, s0, s1

    def _call(self, name: str, step: PagedStep, *args) -> None:
        if step.device != self.device:
            raise ValueError(f"paged cache: a step on {step.device} for a pool on {self.device}")
        if self._at is None:
            raise RuntimeError(f"pool on {self.device}: the sequence kernels run on CUDA only (no CPU fallback)")
        function = getattr(S.lib(), name)
        if torch._C._cuda_getDevice() == self.device.index:
            rc = function(*args, S.stream_ptr())
        else:
            with torch.cuda.device(self.device):
                rc = function(*args, S.stream_ptr())
        if rc:
            S.check(rc, name)

    def write(self, k: torch.Tensor, v: torch.Tensor, step: PagedStep) -> None:
        """The step's keys [rows, kv_heads, dim] and values [rows, kv_heads, vdim] into the pool.  Rows behind the step's last sequence are not looked at.
        Two rows of one step must not have the same place (a page in two sequences' tables, both writing there)."""
        k, k0, k1 = self._rows(k, self.kv_heads, self.dim, step, "keys")
        v, v0, v1 = self._rows(v, self.kv_heads, self.vdim, step, "values")
        self._call("b2l_seq_paged_write", step, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, *(self._at or ()), *(step._at or ()), min(k.shape[0], v.shape[0]), step.seqs, *self._sizes)

    def read(self, step: PagedStep) -> Tuple[torch.Tensor, torch.Tensor]:
        """The rows that `write` with this step puts into the pool, as they lie there: keys [rows, kv_heads, dim] and values in the activation type; zeros where the
        step's tensors have no sequence for a row."""
        G, K, V = self.kv_heads, self.dim, self.vdim
        make = self._like.new_empty if step.seqs else self._like.new_zeros
        k, v = make((step.rows, G, K)), make((step.rows, G, V))
        self._call("b2l_seq_paged_read", step, k.data_ptr(), G * K, K, v.data_ptr(), G * V, V, *(self._at or ()), *(step._at or ()), step.rows, step.seqs, *self._sizes)
        return k, v

    def attend(self, q: torch.Tensor, step: PagedStep, *, scale: Optional[float] = None, window: int = 0, first: int = 0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal softmax attention of the step's tokens (already written) over their sequences:

            out[r, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q[r, h] . k_j), j <= p and (window == 0 or j > p - window or j < first)

        q [rows, heads, dim] with heads a multiple of kv_heads (head h reads key/value head h // (heads / kv_heads)), p the position of row r; scale
        dim^-1/2 unless given.  Returns [rows, heads, vdim] (`out`, contiguous, where given); rows of no sequence, behind the step's last one or before its first,
        are zeros, or as they were in `out`."""
        q, s0, s1 = self._rows(q, 0, self.dim, step, "queries")
        rows, heads, _ = q.shape
        plan = step._plans.get((rows, heads, scale, window, first, self._sizes))
        if plan is None:
            plan = self._plan(rows, heads, scale, window, first, step)
        floats, sizes = plan
        name = "b2l_seq_paged_attention"
        if out is None:
            out, name = (q.new_empty if step.seqs else q.new_zeros)((rows, heads, self.vdim)), "b2l_seq_paged_attention_all"      # which rows have a sequence is known on the device only
        elif out.shape != (rows, heads, self.vdim) or out.dtype != self.dtype or out.device != self.device or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError(f"paged cache: out must be {(rows, heads, self.vdim)} {self.dtype} on {self.device}, contiguous and 16-byte aligned")
        work = step._tensors[1].new_empty((floats,)) if floats else None          # four bytes an entry
        self._call(name, step, q.data_ptr(), s0, s1, *(self._at or ()), *(step._at or ()), out.data_ptr(), work.data_ptr() if floats else None, floats, *sizes)
        return out

    def _plan(self, rows: int, heads: int, scale: Optional[float], window: int, first: int, step: PagedStep) -> tuple:
        """(floats of work space, arguments that are the same in every layer of the step); kept with the step."""
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"paged cache: {heads} query heads over {self.kv_heads} key/value heads")
        if window < 0 or first < 0:
            raise ValueError("paged cache: a negative window or number of first tokens")
        places = step.table.shape[1] * self.page                            # positions below it
        if window >= places or first >= places:
            window = 0                                                      # nothing is hidden
        if not window:
            first = 0
        sizes = (heads, self.kv_heads, self.dim, self.vdim, window, first)
        hints = (step.max_new, step.max_length) + self._codes
        floats = S.lib().b2l_seq_paged_attention_work(rows, step.seqs, step.table.shape[1], self.page, *sizes, *hints)
        plan = (floats, (rows, step.seqs, self.n_pages, self.page) + sizes + (float(self.dim ** -0.5 if scale is None else scale),) + hints)
        step._plans[(rows, heads, scale, window, first, self._sizes)] = plan
        return plan
