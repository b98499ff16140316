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

Several continuations of a sequence, drafted tokens that form a tree or beams:

    PagedTree    the parents of a step's tokens: what each of them sees (for `attend`), and which are accepted
    PagedLayers  the pools of all layers: pages copied, accepted rows moved together
    PagePool     `fork`, `reorder`, `own`, `compact`: pages that sequences share are counted, and say which pages have to be copied

        step = pool.step([("b", 4)])                           # the last token and three drafts: two that follow it, one that follows the first of these
        tree = PagedTree(step, torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda"))
        out = caches[i].attend(q, step, tree=tree)
        kept, counts, following = tree.accept(logits, tokens)
        layers.keep(step, kept, counts)
        pool.take_back("b", 4 - int(counts[0]))
        layers.copy(pool.fork("b", "c"))                       # c goes on from where b stands

A token's key and value rows are quantised by themselves, per head: scale = max(max |x| (1 / c), 2^-126), code = round(x / scale), c = 448 (fp8, e4m3) or 127
(int8).  A row that holds an infinity or NaN reads back as NaN.  A row whose weights sum to zero (it sees no key) attends to zeros.  Everything
is a kernel of libb200seq (include/b2l_seq.h); CUDA only, no CPU fallback, no derivatives."""
import ctypes as C
from typing import Dict, Hashable, List, Mapping, Optional, Sequence, Tuple, Union
from weakref import WeakSet

import torch

from . import _seqlib as S
from .state import PagesFull

STORES = {"act": S.STORE_ACT, "fp8": S.STORE_E4M3, "int8": S.STORE_INT8}
PAGES = (16, 32, 64, 128, 256)
ACTS = (torch.bfloat16, torch.float32)


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
        self._known: Optional[Tuple[int, Optional[int]]] = None             # the most new tokens of a sequence, and the version of `starts` that has them
        self._trees: Optional[WeakSet] = None                               # of `PagedTree`, whose masks are as wide as was needed when they were made

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
        # (.data: `starts` has a version of its own, which tells when it is written over)
        step = cls(both.data[:n + 1], both[n + 1:2 * n + 1], both[2 * n + 1:].view(n, width), rows=rows,
                   max_new=max((new for new, _, _ in sequences), default=0), max_length=max(lengths, default=0))
        step._know(step.max_new)
        return step

    def _know(self, nodes: int) -> None:
        starts = self._tensors[0]
        self._known = (nodes, None if starts.is_inference() else starts._version)

    def _nodes(self) -> int:
        """No sequence has more new tokens than this, whatever the hints: all rows, unless the step was made from the host and not written over since."""
        starts = self._tensors[0]
        if self._known is not None and (starts.is_inference() or starts._version == self._known[1]):
            return self._known[0]
        return self.rows

    def refill(self, other: "PagedStep") -> None:
        """The other step's sequences in this one's tensors (of the same number of sequences and rows, and at least its width), for a graph that was
        recorded with this one."""
        if other.seqs != self.seqs or other.rows != self.rows or other.table.shape[1] > self.table.shape[1]:
            raise ValueError(f"paged step: {other.seqs} sequences with {other.rows} rows and {other.table.shape[1]} pages do not fit {self.seqs} with {self.rows} and {self.table.shape[1]}")
        nodes = other._nodes()
        for tree in self._trees or ():
            if nodes > 32 * tree.words:
                raise ValueError(f"paged step: sequences of up to {nodes} new tokens, the masks of a tree have {32 * tree.words}: it needs `nodes` when it is made")
        self.starts.copy_(other.starts, non_blocking=True)
        self.lengths.copy_(other.lengths, non_blocking=True)
        self.table[:, :other.table.shape[1]].copy_(other.table, non_blocking=True)
        self.table[:, other.table.shape[1]:].fill_(-1)
        self._know(nodes)


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
        self._shared: Dict[int, int] = {}                                   # pages that more than one sequence has -> how many

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
        held = len({p for rid in live for p in self._pages.get(rid, ()) if p >= 0})
        held -= sum(rid in self._pages and self._partial(rid) in self._shared for rid in live)      # another takes that page's place
        return len(self._free) + held >= sum(self.most_pages(n, portion) for n in live.values()) + self.most_pages(tokens, portion)

    def _give(self, page: int) -> None:
        """One sequence no longer has the page: it is free where no other has it."""
        n = self._shared.get(page, 1)
        if n == 1:
            self._free.append(page)
        elif n == 2:
            del self._shared[page]
        else:
            self._shared[page] = n - 1

    def release(self, request_id: Hashable) -> None:
        for p in reversed(self._pages.pop(request_id)):
            if p >= 0:
                self._give(p)
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
        for p in reversed(pages[keep:]):
            if p >= 0:
                self._give(p)
        del pages[keep:]

    # ------------------------------------------------------------------ pages that sequences share
    def _partial(self, request_id: Hashable) -> int:
        """The page that the sequence's next token lies in, or -1 where that begins one (or the page was given back)."""
        return self._pages[request_id][-1] if self._length[request_id] % self.page else -1

    def fork(self, source: Hashable, request_id: Hashable) -> List[Tuple[int, int]]:
        """A new sequence with the tokens of `source`, which stays.  They share the full pages; the one that both go on writing the new one gets a copy of: returns
        the pages to be copied, (from, to), for `PagedLayers.copy` before either sequence's next step.  Raises PagesFull, with nothing changed."""
        if request_id in self._pages:
            raise ValueError(f"page pool: {request_id!r} is a sequence already")
        return self.reorder({request_id: source})

    def reorder(self, sources: Mapping[Hashable, Hashable]) -> List[Tuple[int, int]]:
        """Every sequence of `sources` (new ones too) becomes one with the tokens that its source had before the call; others stay.  What a sequence had is given
        back where no other goes on from it.  Returns the pages to be copied, (from, to), for `PagedLayers.copy` before the next step: none is copied that only one
        sequence goes on writing.  Raises PagesFull, with nothing changed."""
        for s in sources.values():
            if s not in self._pages:
                raise KeyError(f"page pool: no sequence {s!r}")
        keeps: Dict[Hashable, Hashable] = {}                                # source -> the sequence that goes on with its last page
        for s in sources.values():
            if s not in sources or sources[s] == s:
                keeps[s] = s
        for rid, s in sources.items():
            keeps.setdefault(s, rid)
        pages = {rid: list(self._pages[s]) for rid, s in sources.items()}
        copied = [rid for rid, s in sources.items() if keeps[s] != rid and self._partial(s) >= 0]
        for rid in copied:
            pages[rid][-1] = -2                                             # to come
        count: Dict[int, int] = {}
        for rid in set(self._pages) | set(pages):
            for p in pages.get(rid, self._pages.get(rid, ())):
                if p >= 0:
                    count[p] = count.get(p, 0) + 1
        had = [p for rid in sources if rid in self._pages for p in self._pages[rid] if p >= 0]
        free = self._free + [p for p in dict.fromkeys(reversed(had)) if p not in count]
        if len(copied) > len(free):
            raise PagesFull(f"{len(copied)} pages are needed, {len(free)} of {self.n_pages} would be free")
        pairs, lengths = [], {rid: self._length[s] for rid, s in sources.items()}
        for rid in copied:
            pages[rid][-1] = free.pop()
            count[pages[rid][-1]] = 1
            pairs.append((self._partial(sources[rid]), pages[rid][-1]))
        self._free, self._shared = free, {p: n for p, n in count.items() if n > 1}
        self._pages.update(pages)
        self._length.update(lengths)
        return pairs

    def own(self, request_id: Hashable) -> List[Tuple[int, int]]:
        """A copy of the page that the sequence goes on writing where others have it too (after `take_back` into a page that was full when it was shared): the pages
        to be copied, (from, to)."""
        page = self._partial(request_id)
        if page not in self._shared:
            return []
        if not self._free:
            raise PagesFull(f"a page is needed, none of {self.n_pages} is free")
        to = self._free.pop()
        self._pages[request_id][-1] = to
        self._give(page)
        return [(page, to)]

    def compact(self) -> List[Tuple[int, int]]:
        """All sequences' pages among the first ones, as many as there are: the pages to be copied, (from, to), for `PagedLayers.copy` before the next step.  Steps
        that were booked before have the old places."""
        used = {p for pages in self._pages.values() for p in pages if p >= 0}
        to = [p for p in range(len(used)) if p not in used]
        moved = dict(zip(sorted(p for p in used if p >= len(used)), to))
        for pages in self._pages.values():
            pages[:] = [moved.get(p, p) for p in pages]
        self._shared = {moved.get(p, p): n for p, n in self._shared.items()}
        self._free = list(range(self.n_pages - 1, len(used) - 1, -1))
        return list(moved.items())

    def _behind(self, request_id: Hashable) -> List[int]:
        """Places in the sequence's table that no later token sees."""
        if not self.window or request_id not in self._pages:
            return []
        reach = self._length[request_id] - self.window + 1                  # the first position that the next token's window has
        return [i for i, p in enumerate(self._pages[request_id]) if p >= 0 and i * self.page >= self.first and (i + 1) * self.page <= reach]

    def step(self, entries: Sequence[Tuple[Hashable, int]], *, width: int = 0) -> PagedStep:
        """Books `n` more tokens for every (request id, n); ids that are not known begin a sequence.  Raises PagesFull, with nothing booked, where the
        pages do not suffice.  A sequence does not write into a page that others have too: `own` gives it a copy first."""
        if len({rid for rid, _ in entries}) < len(entries):
            raise ValueError("page pool: a request comes twice in one step")
        if any(n < 0 for _, n in entries):
            raise ValueError("page pool: a negative number of tokens")
        behind, new = {rid: self._behind(rid) for rid, _ in entries}, {rid for rid, _ in entries if rid not in self._pages}
        need = sum(max(0, -(-(self._length.get(rid, 0) + n) // self.page) - len(self._pages.get(rid, ()))) for rid, n in entries)
        for rid, n in entries:
            if n and rid in self._pages and self._partial(rid) in self._shared:
                raise ValueError(f"page pool: {rid!r} would write into a page that others have too: it needs one of its own first")
        given: Dict[int, int] = {}
        for rid, places in behind.items():
            for i in places:
                given[self._pages[rid][i]] = given.get(self._pages[rid][i], 0) + 1
        if need > len(self._free) + sum(n == self._shared.get(p, 1) for p, n in given.items()):
            raise PagesFull(f"{need} pages are needed, {len(self._free)} of {self.n_pages} are free")
        sequences = []
        for rid, _ in entries:
            for i in behind[rid]:
                self._give(self._pages[rid][i])
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


def _launch(device: torch.device, name: str, *args) -> None:
    """A kernel on the device, whichever is the current one."""
    if device.type != "cuda":
        raise RuntimeError(f"tensors on {device}: the sequence kernels run on CUDA only (no CPU fallback)")
    function = getattr(S.lib(), name)
    if torch._C._cuda_getDevice() == device.index:
        rc = function(*args, S.stream_ptr())
    else:
        with torch.cuda.device(device):
            rc = function(*args, S.stream_ptr())
    if rc:
        S.check(rc, name)


def _whole(what: str, x: torch.Tensor, dtype: torch.dtype, device: torch.device, entries: int) -> torch.Tensor:
    """x, of at least so many entries one behind the other."""
    if x.dtype != dtype or x.dim() != 1 or x.shape[0] < entries or x.device != device or (x.shape[0] > 1 and x.stride(0) != 1):
        raise ValueError(f"{what} {tuple(x.shape)} {x.dtype} on {x.device}: [{entries}] {dtype} on {device}, consecutive, is wanted")
    return x


def _matrix(x: torch.Tensor, columns: int) -> Tuple[torch.Tensor, int]:
    """x [rows, columns] with its rows' entries consecutive (else a copy), and the entries between its rows."""
    s0, s1 = x.stride()
    if x.shape[0] <= 1:
        s0 = columns
    if (s1 != 1 and columns > 1) or s0 < columns:
        return x.contiguous(), columns
    return x, s0


class PagedTree:
    """The new tokens of a step as trees: parents[r] (int32 [rows], on the device) is the place, among its sequence's new tokens, of the token that row r follows,
    one before it, or -1 where it follows the sequence as it was.  A token is at the position of its parent and one more (`positions`, int32 [rows], for the rotation of
    queries and keys); keys and values lie in the order of the rows all the same.

    `attend(.., tree=tree)` lets a token see what was there before the step, its ancestors and itself: the bits of `masks` (int32 [rows, words], bit i of a row for new
    token i), which may be written over to see others.  `window` and `first`, those of `attend`, hide ancestors out of reach.  `nodes`: the most new tokens that a
    sequence of the step ever has, by default the most that one has now (of a step that was made from tensors, all of its rows, as `max_new` is a hint).

    The step's tensors and `parents` may be overwritten between replays of a graph that was recorded with them; then `update` belongs into the graph too.  Where a
    sequence may get more new tokens by that than one has now, `nodes` has to say so: tokens from 32 `words` on are not seen (`PagedStep.refill` refuses them)."""

    def __init__(self, step: PagedStep, parents: torch.Tensor, *, nodes: int = 0, window: int = 0, first: int = 0) -> None:
        self.step, self.device = step, step.device
        self.parents = _whole("paged tree: parents", parents, torch.int32, step.device, step.rows)
        if nodes < 0 or window < 0 or first < 0:
            raise ValueError("paged tree: a negative number of tokens, window or number of first tokens")
        self.words = max(1, -(-(int(nodes) or step._nodes()) // 32))
        self.window, self.first = min(int(window), 2 ** 30), min(int(first), 2 ** 30)
        make = step.starts.new_empty if step.seqs else step.starts.new_zeros
        self.masks, self.depths, self.positions = make((step.rows, self.words)), make((step.rows,)), make((step.rows,))
        self._works: Dict[int, int] = {}                                    # bytes of work space of `accept`, by the vocabulary
        if step._trees is None:
            step._trees = WeakSet()
        step._trees.add(self)
        self.update()

    def update(self) -> None:
        """masks, depths and positions from the parents and the step as they are now."""
        s = self.step
        _launch(self.device, "b2l_seq_tree_build", self.parents.data_ptr(), s.starts.data_ptr(), s.lengths.data_ptr(), self.masks.data_ptr(), self.words, self.depths.data_ptr(),
                self.positions.data_ptr(), s.rows, s.seqs, self.window, self.first)

    def accept(self, logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 0.0,
               noise: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Which of the step's tokens (int32 or int64 [rows]) the model would have chosen itself.  A row's target is the largest of its logits ([rows, vocab], bf16 or
        f32), with a temperature one drawn from softmax(logits / temperature): the largest of logits / temperature - log noise, the noise (f32 [rows, vocab]) drawn from
        Exp(1) unless given.  From a sequence's first new token (which is taken) the path goes to a child whose token is its parent's target as long as there is one; so
        the tokens of the path and the last one's target are what step after step without drafts gives.

        Returns int32 tensors: kept [rows], the places of the path's tokens among the sequence's new ones, -1 behind them; counts [sequences], how many; following
        [sequences], the last one's target (-1 for a sequence without new tokens)."""
        s, rows, shape = self.step, self.step.rows, logits.shape
        if len(shape) != 2 or shape[0] < rows or shape[1] < 1 or logits.device != self.device or logits.dtype not in ACTS:
            raise ValueError(f"paged tree: logits {tuple(shape)} {logits.dtype} on {logits.device}, [{rows}, vocab] in bf16 or f32 on {self.device} are wanted")
        wide = tokens.dtype == torch.int64
        tokens = _whole("paged tree: tokens", tokens, torch.int64 if wide else torch.int32, self.device, rows)
        if not 0.0 <= temperature < float("inf"):
            raise ValueError(f"paged tree: a temperature of {temperature}")
        vocab = shape[1]
        logits, ld = _matrix(logits, vocab)
        ldn, at = vocab, None
        if temperature > 0.0:
            if noise is None:
                noise = torch.empty((rows, vocab), dtype=torch.float32, device=self.device).exponential_(1)
            if noise.dtype != torch.float32 or noise.dim() != 2 or noise.shape[0] < rows or noise.shape[1] != vocab or noise.device != self.device:
                raise ValueError(f"paged tree: noise {tuple(noise.shape)} {noise.dtype} on {noise.device}, [{rows}, {vocab}] in f32 on {self.device} is wanted")
            noise, ldn = _matrix(noise, vocab)
            at = noise.data_ptr()
        size = self._works.get(vocab)
        if size is None:
            size = self._works[vocab] = S.lib().b2l_seq_tree_accept_work(rows, vocab)
        starts, seqs = s._tensors[0], s.seqs
        whole = -(-size // 4)                                               # one allocation for all, the work space first: it is aligned
        work, kept, counts, following = starts.new_empty(whole + rows + 2 * seqs).split_with_sizes([whole, rows, seqs, seqs])
        if not seqs:
            kept.fill_(-1)
        _launch(self.device, "b2l_seq_tree_accept", logits.data_ptr(), ld, at, ldn, float(temperature), self.parents.data_ptr(), starts.data_ptr(), tokens.data_ptr(), int(wide),
                kept.data_ptr(), counts.data_ptr(), following.data_ptr(), work.data_ptr(), size, rows, seqs, vocab, S.act_code(logits.dtype))
        return kept, counts, following


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
               out: Optional[torch.Tensor] = None, tree: Optional[PagedTree] = None) -> torch.Tensor:
        """Causal softmax attention of the step's tokens (already written) over their sequences:

            out[r, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q[r, h] . k_j), j <= p and (window == 0 or j > p - window or j < first)

        q [rows, heads, dim] with heads a multiple of kv_heads (head h reads key/value head h // (heads / kv_heads)), p the position of row r; scale
        dim^-1/2 unless given.  Returns [rows, heads, vdim] (`out`, contiguous, where given); rows of no sequence, behind the step's last one or before its first,
        are zeros, or as they were in `out`.

        With a `tree` of the step, p is the token's position in it, and of the step's new tokens a row sees those that the tree says, whatever the window: `window` and
        `first` hide what was there before the step, and the tree hides ancestors by those that it was made with."""
        q, s0, s1 = self._rows(q, 0, self.dim, step, "queries")
        rows, heads, _ = q.shape
        if tree is not None:
            return self._attend_tree(q, s0, s1, step, tree, scale, window, first, out)
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

    def _attend_tree(self, q: torch.Tensor, s0: int, s1: int, step: PagedStep, tree: PagedTree, scale: Optional[float], window: int, first: int,
                     out: Optional[torch.Tensor]) -> torch.Tensor:
        if tree.step is not step:
            raise ValueError("paged cache: the tree of another step")
        rows, heads = step.rows, q.shape[1]                                 # masks are of these
        shape = (q.shape[0], heads, self.vdim)
        plan = step._plans.get((rows, heads, scale, window, first, self._sizes, True))
        if plan is None:
            plan = self._plan(rows, heads, scale, window, first, step, True)
        floats, sizes = plan
        zeros = out is None
        if zeros:
            out = (q.new_empty if step.seqs else q.new_zeros)(shape)
            if shape[0] > rows:
                out[rows:].zero_()
        elif out.shape != shape or out.dtype != self.dtype or out.device != self.device or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError(f"paged cache: out must be {shape} {self.dtype} on {self.device}, contiguous and 16-byte aligned")
        work = step._tensors[1].new_empty((floats,)) if floats else None
        self._call("b2l_seq_paged_attention_tree", step, q.data_ptr(), s0, s1, *(self._at or ()), *(step._at or ()), tree.masks.data_ptr(), tree.words, tree.depths.data_ptr(), int(zeros),
                   out.data_ptr(), work.data_ptr() if floats else None, floats, *sizes)
        return out

    def _plan(self, rows: int, heads: int, scale: Optional[float], window: int, first: int, step: PagedStep, tree: bool = False) -> tuple:
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
        work = S.lib().b2l_seq_paged_attention_tree_work if tree else S.lib().b2l_seq_paged_attention_work
        with torch.cuda.device(self.device if self.device.type == "cuda" else -1):      # its SMs decide how keys are split
            floats = work(rows, step.seqs, step.table.shape[1], self.page, *sizes, *hints)
        plan = (floats, (rows, step.seqs, self.n_pages, self.page) + sizes + (float(self.dim ** -0.5 if scale is None else scale),) + hints)
        step._plans[(rows, heads, scale, window, first, self._sizes) + ((True,) if tree else ())] = plan
        return plan


class PagedLayers:
    """The pools of all of a model's layers, alike in sizes and types, whose pages are moved together."""

    def __init__(self, caches: Sequence[PagedCache]) -> None:
        self.caches = list(caches)
        if not self.caches:
            raise ValueError("paged layers: no pool")
        one = self.caches[0]
        if any(c._sizes != one._sizes or c.device != one.device for c in self.caches):
            raise ValueError("paged layers: pools of different sizes or types, or on different devices")
        self.device = one.device
        self._sizes = one._sizes
        flat = [a or 0 for c in self.caches for a in (c._at or (0, 0, 0, 0))]
        self._at = (C.c_void_p * len(flat))(*flat)

    def copy(self, pages: Union[torch.Tensor, Sequence[Tuple[int, int]]]) -> None:
        """Pages of every layer: (from, to) of each, from the host or as int32 [n, 2] on the device.  No page comes twice as `to`, and none as both.  Pairs with a page
        outside the pool are left out."""
        if not isinstance(pages, torch.Tensor):
            pages = list(pages)
            if any(not 0 <= p < self._sizes[0] for pair in pages for p in pair):
                raise ValueError(f"paged layers: pages outside the pool of {self._sizes[0]}")
            targets = {b for _, b in pages}
            if len(targets) < len(pages) or targets & {a for a, _ in pages}:
                raise ValueError("paged layers: a page that is written twice, or copied and written")
            if not pages:
                return
            pages = torch.tensor(pages, dtype=torch.int32).to(self.device)
        if pages.dtype != torch.int32 or pages.dim() != 2 or pages.shape[1] != 2 or pages.device != self.device or not pages.is_contiguous():
            raise ValueError(f"paged layers: pages {tuple(pages.shape)} {pages.dtype} on {pages.device}: [n, 2] int32 on {self.device}, contiguous, is wanted")
        if pages.data_ptr() % 8:
            pages = pages.clone()
        _launch(self.device, "b2l_seq_paged_copy", C.addressof(self._at), len(self.caches), pages.data_ptr(), pages.shape[0], *self._sizes)

    def keep(self, step: PagedStep, kept: torch.Tensor, counts: torch.Tensor) -> None:
        """Of a step's new tokens those of a path (as `PagedTree.accept` returns them: kept int32 [rows], ascending for every sequence, counts int32 [sequences]) moved
        together in every layer: behind the tokens that the sequence had before the step.  `PagePool.take_back` gives the other tokens' places back.
        Between the step and this none of its sequences is forked: their pages are written."""
        kept = _whole("paged layers: kept", kept, torch.int32, self.device, step.rows)
        counts = _whole("paged layers: counts", counts, torch.int32, self.device, step.seqs)
        if step.device != self.device:
            raise ValueError(f"paged layers: a step on {step.device} for pools on {self.device}")
        pages, page, *sizes = self._sizes
        _launch(self.device, "b2l_seq_paged_keep", C.addressof(self._at), len(self.caches), *(step._at or (None, None, None, 1, 1)), kept.data_ptr(), counts.data_ptr(), step.rows,
                step.seqs, pages, page, *sizes)
