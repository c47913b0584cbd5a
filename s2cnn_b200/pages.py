"""Kept keys and values of growing sequences in pages of one pool: sequences take pages as they grow, share those of a common
beginning, and give them back.

* ``norm_rotate_store`` writes the keys (normed and turned, see ``sequence.norm_rotate``) and values of new positions to their pages;
* ``paged_attention`` is ``sequence.attention`` for new positions over what is kept there;
* ``copy_pages`` copies pages within their pool;
* ``PagedCache`` holds the pool and says which pages are whose: ``extend``, ``fork``, ``truncate``, ``free``, ``compact``.

The reference has no counterpart.  Keys and values are [pages, positions of a page, kv_heads, dim] (any strides with a contiguous last
axis); position j of sequence n lies in page ``pages[n, j // page]``, at ``j % page``.  The positions of a page are a power of two, at
least 8.  An entry that is no page of the pool is not written, and reads as NaN.  None of these has a gradient: a call that
autograd would record is refused.
"""
import torch

from .ops import cuda_ops


def norm_rotate_store(q, k, v, keys, values, pages, frequencies=None, q_weight=None, k_weight=None, eps=None, positions=0, lengths=None, interleaved=False,
                      magnitude=1.0):
    """``sequence.norm_rotate`` of new queries and keys with the keys, and the values as they are, written to their pages in the
    same pass.

    :param q: [batch, new, heads, dim], or None: keys and values alone
    :param k, v: [batch, new, kv_heads, dim]
    :param keys, values: [pages, positions of a page, kv_heads, dim], written in place
    :param pages: int32 [batch, columns], the pages of each sequence
    :param positions: of the rows, as in ``norm_rotate``; they are the places among the kept ones, too.  No two rows of a call may have
        one place (it holds either then, or parts of both)
    :param lengths: int32 [batch], the rows that are filled (None: all); what is beyond them is neither read nor written
    :return: the normed and turned queries; 0 beyond ``lengths``, NaN where the position has no page.  None without q
    """
    start, positions = (0, positions) if isinstance(positions, torch.Tensor) else (positions, None)
    return cuda_ops().norm_rotate_store(q, k, v, keys, values, pages, frequencies, q_weight, k_weight, positions, lengths, _eps(eps), int(start),
                                        bool(interleaved), float(magnitude))


def _eps(eps):
    assert eps is None or eps >= 0, "eps is negative"
    return -1.0 if eps is None else float(eps)


def paged_attention(q, keys, values, pages, bias=None, buckets=None, causal=False, scale=None, q_start=0, q_lengths=None, kv_lengths=None):
    """``sequence.attention`` (its formula and its other parameters) over keys and values in pages: for new positions, whose keys and
    values are read once, or, beyond 16 rows of queries and heads per key head, once for every 16.

    Beyond 128 rows (256 in float32) they are first copied into one array, where the whole of their columns takes at most 1 GB for
    one sequence, whatever is kept, for the kernels of ``attention``, which round bfloat16 weights to 8 bits; otherwise these have 16 (and
    the float32 ones 22: products of two TF32 parts).

    :param q: [batch, queries, heads, dim], dim <= 128; any strides with a contiguous last axis
    :param keys, values: [pages, positions of a page, kv_heads, dim]
    :param pages: int32 [batch, columns], the pages of each sequence
    :param kv_lengths: int32 [batch], the positions that are kept (None: all of the columns')
    :return: [batch, queries, heads, dim]
    """
    starts = None
    if isinstance(q_start, torch.Tensor):
        q_start, starts = 0, q_start
    if scale is None:
        scale = q.size(-1) ** -0.5
    return cuda_ops().paged_attention(q, keys, values, pages, bias, buckets, starts, q_lengths, kv_lengths, bool(causal), float(scale), int(q_start))


def copy_pages(storage, source, target):
    """Page ``target[i]`` of ``storage`` [pages, ...] (each page contiguous, any type) becomes a copy of page ``source[i]``, in
    place; entries that are no page are left out.

    :param source, target: int32 [n] on the device of the storage.  A page may be the source of several, but no target may occur
        twice or be a source, too: such a page holds a mixture afterwards
    """
    cuda_ops().copy_pages(storage, source, target)


class PagedCache:
    """The kept keys and values of up to ``sequences`` sequences, in all layers of a model, in a pool of ``pages`` pages.

    ``columns`` are the pages that a sequence can have: by default, all of the pool, up to 2^28 positions.  Long first passes want them no
    larger than needed (see ``paged_attention``); ``table[:, :n].contiguous()`` does for a call on sequences that are known to be short.

    ``storage`` [pages, layers, 2, kv_heads, page, dim rounded up to 16 bytes] has the positions of a head in a page one after
    another, so that attention reads them in whole pieces, and all layers of a page together, so that forking copies one piece.

    Which page is whose is decided on the host, which knows how far each sequence has grown (``lengths``, a list); the
    kernels read ``table`` int32 [sequences, columns] and ``filled`` int32 [sequences] on the device.  These keep their addresses,
    so that a step may be captured and replayed after ``extend`` (the account's own calls are not captured).  Everything runs on the
    current stream; nothing waits for the device.

    A step of a model: ``cache.extend(new)`` makes room for new positions, the layers run ``SequenceBlock.step_pages`` with
    ``cache.keys(layer)``, ``cache.values(layer)``, ``cache.table`` and ``cache.filled`` (the positions before this step), and
    ``cache.advance()`` ends the step.  ``extend`` called again for the same step (it was not advanced) changes what it asks for.
    """

    def __init__(self, pages, page, kv_heads, dim, sequences, columns=None, layers=1, dtype=torch.float32, device="cuda"):
        assert page >= 8 and page & (page - 1) == 0, "PagedCache: the positions of a page are a power of two, at least 8"
        assert pages >= 1 and sequences >= 1 and layers >= 1 and kv_heads >= 1 and dim >= 1
        assert pages * page < 1 << 31, "PagedCache: at most 2^31 positions in a pool"
        step = 16 // torch.empty(0, dtype=dtype).element_size()
        self.page, self.dim, self.layers = page, dim, layers
        self.storage = torch.zeros(pages, layers, 2, kv_heads, page, -(-dim // step) * step, dtype=dtype, device=device)
        columns = min(pages, (1 << 28) // page) if columns is None else columns
        assert columns * page <= 1 << 28, "PagedCache: at most 2^28 positions in a sequence"
        self.table = torch.full((sequences, columns), -1, dtype=torch.int32, device=device)
        self.filled = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.lengths = [0] * sequences
        self._new = [0] * sequences                        # of the step that has begun
        self._pages = [[] for _ in range(sequences)]
        self._uses = [0] * pages                           # sequences that hold a page
        self._free = list(range(pages - 1, -1, -1))

    def keys(self, layer=0):
        """[pages, page, kv_heads, dim]"""
        return self.storage[:, layer, 0].transpose(1, 2)[..., :self.dim]

    def values(self, layer=0):
        return self.storage[:, layer, 1].transpose(1, 2)[..., :self.dim]

    @property
    def free_pages(self):
        return len(self._free)

    def extend(self, new):
        """Begins a step of ``new`` positions for every sequence (a number or one per sequence): pages that they need are taken, and
        a shared page that would be written is copied first.  Raises MemoryError, and changes nothing, if the pool does not hold
        them."""
        self._uncaptured("extend")
        new = [new] * len(self.lengths) if isinstance(new, int) else list(new)
        assert len(new) == len(self.lengths) and min(new) >= 0, "extend: a number of new positions for each sequence"
        need, copies = {}, []
        uses = {}                                          # of shared pages, as this call leaves them
        for s, n in enumerate(new):
            end = self.lengths[s] + n
            columns = -(-end // self.page)
            if columns > self.table.size(1):
                raise MemoryError("PagedCache: sequence %d would have %d positions, more than %d columns hold" % (s, end, self.table.size(1)))
            if n and self.lengths[s] % self.page:
                last = self._pages[s][self.lengths[s] // self.page]
                if uses.get(last, self._uses[last]) > 1:
                    copies.append((s, last))
                    uses[last] = uses.get(last, self._uses[last]) - 1
            if columns > len(self._pages[s]):
                need[s] = columns - len(self._pages[s])
        if len(copies) + sum(need.values()) > len(self._free):
            raise MemoryError("PagedCache: %d more pages are needed, %d are free" % (len(copies) + sum(need.values()), len(self._free)))
        moved, entries = [], []
        for s, last in copies:
            own, column = self._take(), self.lengths[s] // self.page
            self._uses[last] -= 1
            self._pages[s][column] = own
            moved.append((last, own))
            entries.append((s, column, own))
        for s, n in need.items():
            for _ in range(n):
                entries.append((s, len(self._pages[s]), self._take()))
                self._pages[s].append(entries[-1][2])
        self._copy(moved)
        self._upload(entries)
        self._new = new

    def advance(self):
        """Ends the step: its positions count as filled."""
        self._uncaptured("advance")
        if any(self._new):
            self.lengths = [a + b for a, b in zip(self.lengths, self._new)]
            self._new = [0] * len(self.lengths)
            self.filled.copy_(self._staged(torch.tensor(self.lengths, dtype=torch.int32)), non_blocking=True)

    def fork(self, source, target):
        """Sequence ``target``, which is empty, continues from all that is filled of ``source``: its pages are shared until one of
        the two writes to the last of them."""
        self._settled("fork")
        assert source != target and not self._pages[target] and self.lengths[target] == 0, "fork: the target is not empty"
        self._pages[target] = self._pages[source][:-(-self.lengths[source] // self.page)]
        for p in self._pages[target]:
            self._uses[p] += 1
        self._upload([(target, column, p) for column, p in enumerate(self._pages[target])])
        self._grown(target, self.lengths[source])

    def truncate(self, sequence, length):
        """Forgets the positions of a sequence from ``length`` on."""
        self._settled("truncate")
        assert 0 <= length <= self.lengths[sequence], "truncate: the sequence is shorter"
        keep = -(-length // self.page)
        for p in self._pages[sequence][keep:]:
            self._give(p)
        self._upload([(sequence, column, -1) for column in range(keep, len(self._pages[sequence]))])
        del self._pages[sequence][keep:]
        self._grown(sequence, length)

    def free(self, sequence):
        """Gives back all pages of a sequence."""
        self.truncate(sequence, 0)

    def compact(self):
        """Moves pages that are held to the front of the pool, shared ones once; returns how many there are."""
        self._settled("compact")
        held = len(self._uses) - len(self._free)
        holes = [p for p in range(held) if not self._uses[p]]
        moved = list(zip([p for p in range(held, len(self._uses)) if self._uses[p]], holes))
        self._copy(moved)
        to = dict(moved)
        for a, b in moved:
            self._uses[b], self._uses[a] = self._uses[a], 0
        self._free = list(range(len(self._uses) - 1, held - 1, -1))
        self._upload([(s, column, to[p]) for s, pages in enumerate(self._pages) for column, p in enumerate(pages) if p in to])
        self._pages = [[to.get(p, p) for p in pages] for pages in self._pages]
        return held

    # -- the host's account
    def _uncaptured(self, what):
        assert not (self.storage.is_cuda and torch.cuda.is_current_stream_capturing()), what + ": the account changes between captured steps, not in one"

    def _settled(self, what):
        self._uncaptured(what)
        assert not any(self._new), what + ": a step has begun (advance() ends it)"

    def _take(self):
        p = self._free.pop()
        self._uses[p] = 1
        return p

    def _give(self, p):
        self._uses[p] -= 1
        if not self._uses[p]:
            self._free.append(p)

    def _copy(self, moved):
        if moved:
            which = self._on_device(torch.tensor(moved, dtype=torch.int32).t().contiguous())
            copy_pages(self.storage, which[0], which[1])

    def _grown(self, s, length):
        self.lengths[s] = length
        self.filled[s].fill_(length)

    def _upload(self, entries):
        """the entries (sequence, column, page) of the table that have changed"""
        if entries:
            at, pages = self._on_device(torch.tensor([(s * self.table.size(1) + column, page) for s, column, page in entries]).t().contiguous())
            self.table.view(-1)[at] = pages.int()

    def _staged(self, t):
        # (from pageable memory the driver may wait for the stream before it copies, and does from 64 KB on; a block of the pinned memory that
        # torch keeps is not used again before the copy from it has run)
        return t.pin_memory() if self.storage.is_cuda else t

    def _on_device(self, t):
        return self._staged(t).to(self.storage.device, non_blocking=True)
