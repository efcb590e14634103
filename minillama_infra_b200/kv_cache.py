"""Pages of a key-value cache: who holds which, and when one has to be copied.

`PagedKvCache` owns a cache's memory and its page table.  Sequences are rows of
the page table; a page may belong to several of them (forks), and is copied for
one of them when that one is about to write into it.  The bookkeeping is on the
host; the tensors that the kernels read (`cache`, `page_table`) are on the
device, and every change of them is ordered on the current stream (which must
not be capturing then: RuntimeError).  A token that needs no new page changes
nothing on the device; one that does sends one entry of the page table.

    kv = PagedKvCache(layers=16, pages=4096, kv_heads=8, head_dim=64, max_seqs=64)
    s = kv.new()
    kv.extend([s], [prompt_len])            # slots for the prompt's tokens
    ops.rope_append(q, q, k, v, kv.cache, layer, pos, kv.page_table, turns, seq=...)
    t = kv.fork(s)                          # shares every page
    kv.extend([s, t])                       # one more token each: t's (or s's) last page is copied
    kv.free(s); kv.compact()
"""
from __future__ import annotations

from array import array

from . import ops

__all__ = ["PagedKvCache"]


class PagedKvCache:
    """layout "heads" keeps a page's slots of one head together (16-bit heads of
    64 then make runs of page_size * 128 bytes), "tokens" a token's heads."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, page_size: int = 16,
                 max_seqs: int = 64, max_pages: int | None = None, dtype=None, device="cuda",
                 layout: str = "heads"):
        import torch

        if layout not in ("heads", "tokens"):
            raise ValueError("layout: heads or tokens")
        max_pages = pages if max_pages is None else max_pages
        if min(layers, pages, kv_heads, head_dim, page_size, max_seqs, max_pages) <= 0:
            raise ValueError("sizes have to be positive")
        dtype = torch.bfloat16 if dtype is None else dtype
        inner = (kv_heads, page_size) if layout == "heads" else (page_size, kv_heads)
        k, v = (torch.zeros((layers, pages, *inner, head_dim), dtype=dtype, device=device) for _ in range(2))
        if layout == "tokens":
            k, v = k.transpose(2, 3), v.transpose(2, 3)
        self.cache = ops.KvCache(k, v)
        self.page_size, self.max_pages = page_size, max_pages
        # -1 names no page: a kernel that is led there reports it
        self.page_table = torch.full((max_seqs, self.max_pages), -1, dtype=torch.int32, device=device)
        self._free_pages = list(range(pages - 1, -1, -1))
        self._free_rows = list(range(max_seqs - 1, -1, -1))
        self._holders = [0] * pages
        self._pages: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}

    @property
    def free_pages(self) -> int:
        return len(self._free_pages)

    def length(self, seq: int) -> int:
        return self._lengths[seq]

    def pages(self, seq: int) -> list[int]:
        return list(self._pages[seq])

    def new(self) -> int:
        """An empty sequence: its row of the page table."""
        if not self._free_rows:
            raise MemoryError("every row of the page table is in use")
        seq = self._free_rows.pop()
        self._pages[seq], self._lengths[seq] = [], 0
        return seq

    def extend(self, seqs, counts=None) -> None:
        """Slots for counts[i] (one) more tokens of seqs[i].  All or nothing: without
        pages enough, MemoryError, and nothing has changed; nor has it when a copy
        or an update of the page table raises (every method keeps to that)."""
        seqs = list(seqs)
        counts = [1] * len(seqs) if counts is None else list(counts)
        if len(counts) != len(seqs) or len(set(seqs)) != len(seqs) or any(n < 0 for n in counts):
            raise ValueError("expected distinct sequences and a count >= 0 for each")
        # how many hold each page, as the copies below change it
        holders = {p: self._holders[p] for s in seqs for p in self._pages[s][-1:]}
        copies, more = [], []
        for seq, n in zip(seqs, counts):
            have, length = self._pages[seq], self._lengths[seq]
            want = -(-(length + n) // self.page_size)
            if want > self.max_pages:
                raise MemoryError(f"sequence {seq}: {length + n} tokens need more than {self.max_pages} pages")
            more.append(want - len(have))
            if n and length % self.page_size and holders[have[-1]] > 1:
                holders[have[-1]] -= 1
                copies.append(seq)
        needed = sum(more) + len(copies)
        if needed > len(self._free_pages):
            raise MemoryError(f"{needed} pages needed, {len(self._free_pages)} free")
        if needed:
            self._grow(seqs, copies, more, needed)
        for seq, n in zip(seqs, counts):
            self._lengths[seq] += n

    def _grow(self, seqs, copies, more, needed) -> None:
        """Copies of the last pages of `copies`, and more[i] new pages for seqs[i]: `needed` in all."""
        pages = self._free_pages[len(self._free_pages) - needed:][::-1]
        moved = [(self._pages[seq][-1], page) for seq, page in zip(copies, pages)]
        rows, cols, at = list(copies), [len(self._pages[seq]) - 1 for seq in copies], len(copies)
        for seq, n in zip(seqs, more):
            if n:
                rows += [seq] * n
                cols += range(len(self._pages[seq]), len(self._pages[seq]) + n)
        # the device first: should it refuse, the pages are still free and the sequences what they were
        self._copy(moved)
        self._write(rows, cols, pages)
        del self._free_pages[len(self._free_pages) - needed:]
        for page in pages:
            self._holders[page] = 1
        for seq, (old, page) in zip(copies, moved):
            self._holders[old] -= 1
            self._pages[seq][-1] = page
        for seq, n in zip(seqs, more):
            self._pages[seq] += pages[at:at + n]
            at += n

    def fork(self, seq: int) -> int:
        """A new sequence that starts with all of seq's tokens and shares its pages."""
        pages, length = list(self._pages[seq]), self._lengths[seq]  # before a row is looked for
        if not self._free_rows:
            raise MemoryError("every row of the page table is in use")
        new = self._free_rows[-1]
        if pages:
            self.page_table[new, :len(pages)] = self._send(pages)[0]
        self._free_rows.pop()
        self._pages[new], self._lengths[new] = pages, length
        for page in pages:
            self._holders[page] += 1
        return new

    def free(self, seq: int) -> None:
        """Gives the sequence's row back, and the pages that no other holds."""
        pages = self._pages[seq]
        self._check_stream()
        self.page_table[seq].fill_(-1)
        del self._pages[seq], self._lengths[seq]
        for page in pages:
            self._holders[page] -= 1
            if not self._holders[page]:
                self._free_pages.append(page)
        self._free_rows.append(seq)

    def compact(self) -> int:
        """Moves pages so that those in use are the first ones; how many moved."""
        used = sum(1 for n in self._holders if n)
        holes = [p for p in range(used) if not self._holders[p]]
        # each move goes from behind `used` to before it: no page is both source and destination
        moved = dict(zip((p for p in range(used, len(self._holders)) if self._holders[p]), holes))
        if not moved:
            return 0
        entries = [(seq, col, moved[page]) for seq, pages in self._pages.items() for col, page in enumerate(pages)
                   if page in moved]
        self._copy(list(moved.items()))
        self._write(*zip(*entries))
        for old, page in moved.items():
            self._holders[page], self._holders[old] = self._holders[old], 0
        for seq, col, page in entries:
            self._pages[seq][col] = page
        self._free_pages = list(range(len(self._holders) - 1, used - 1, -1))
        return len(moved)

    def _check_stream(self) -> bool:
        """Whether the cache is a GPU's.  A change within a capture would be made at its replays, not now."""
        import torch

        on_gpu = self.page_table.device.type == "cuda"
        if on_gpu and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the pages of a cache cannot change while the current stream is capturing")
        return on_gpu

    def _send(self, *lists):
        """Lists of one length as rows of an int32 tensor on the device, by a copy that the host does not wait for."""
        import torch

        on_gpu = self._check_stream()
        numbers = array("i")
        for x in lists:
            numbers.extend(x)
        t = torch.frombuffer(numbers, dtype=torch.int32).view(len(lists), -1)
        return (t.pin_memory() if on_gpu else t).to(self.page_table.device, non_blocking=True)

    def _copy(self, pairs) -> None:
        if pairs:
            ops.kv_copy_pages(self.cache, *self._send(*zip(*pairs)))

    def _write(self, rows, cols, pages) -> None:
        """page_table[rows[i], cols[i]] = pages[i], and no others: a token that crosses into a new page changes one
        entry, however long its sequence."""
        if len(rows) <= 4:  # a fill takes 7 us, sending numbers and an indexed write 36
            self._check_stream()
            for row, col, page in zip(rows, cols, pages):
                self.page_table[row, col].fill_(page)
        else:
            rows, cols, pages = self._send(rows, cols, pages)
            self.page_table[rows, cols] = pages
