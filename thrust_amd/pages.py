"""Pages of a cache: sequences that share pages, grow, fork, end, and are closed up again.

All of it is in device memory and nothing is read back: calls can be captured into a graph, and their
effect depends on the contents of the arrays alone.  A page that no sequence names (refs 0) is free;
requests take the lowest free pages in their order.
"""
import ctypes

import torch

from . import capi, device as dev


class PageCache:
    """`pools`: the arrays that are paged together (a layer's keys, its values, its recurrent states ...),
    each [pages, ...], contiguous, of any type, with the same number of pages and of bytes a page.  A page
    holds `page_size` tokens; for a state, which is never full, any number above the longest sequence.

    tables  int32 [max_sequences, max_pages]  the pages of each sequence, -1 behind them
    lengths int32 [max_sequences]             tokens; the first ceil(length / page_size) entries are held
    refs    int32 [pages]                     how many tables name a page

    They start empty, or are the given ones, which are then used in place; their contents may be written
    between calls, but they are not replaced by others (make a cache with those instead).
    """

    tables = property(lambda self: self._tables)
    lengths = property(lambda self: self._lengths)
    refs = property(lambda self: self._refs)

    def __init__(self, pools, page_size, max_sequences, max_pages, tables=None, lengths=None, refs=None):
        pools = list(pools)
        if not pools:
            raise ValueError("a cache needs a pool")
        device = dev.need_device(*pools, tables, lengths, refs)
        pages = pools[0].shape[0] if pools[0].dim() else -1
        total = pools[0].numel() * pools[0].element_size()
        for p in pools:
            if p.dim() < 1 or p.shape[0] != pages or not p.is_contiguous():
                raise ValueError("pools must be contiguous and of the same number of pages")
            if p.numel() * p.element_size() != total:
                raise ValueError("pools must have the same number of bytes a page")
        if page_size < 1 or max_sequences < 0 or max_pages < 0 or page_size * max_pages > 0x7fffffff:
            raise ValueError("page_size must be positive, and page_size * max_pages below 2^31")
        self.pools, self.page_size, self.device = pools, page_size, device
        self._tables = self._array(tables, (max_sequences, max_pages), -1, "tables")
        self._lengths = self._array(lengths, (max_sequences,), 0, "lengths")
        self._refs = self._array(refs, (pages,), 0, "refs")
        self._home = dev.stream(device)
        self._pointers = dev.Outliving(torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64).to(device), device)
        self._args = capi.PageCacheArgs(pools=self._pointers.tensor.data_ptr(), page_bytes=total // max(pages, 1), num_pools=len(pools), num_pages=pages,
                                        page_size=page_size, num_sequences=max_sequences, max_pages=max_pages,
                                        tables=self.tables.data_ptr(), lengths=self.lengths.data_ptr(), refs=self.refs.data_ptr())
        self._ref = ctypes.byref(self._args)
        self._sizes = {}
        self._own = (self._tables, self._lengths, self._refs)
        self._all = (*self._own, *pools)

    def _array(self, given, shape, value, what):
        if given is None:
            return dev.empty(self.pools[0], shape, torch.int32).fill_(value)
        if given.dtype != torch.int32 or given.shape != shape or not given.is_contiguous():
            raise ValueError(f"{what} must be int32 {list(shape)}, contiguous")
        return given

    def _requests(self, *ids):
        if dev.need_device(*ids) != self.device:
            raise ValueError("tensors on another device than the cache")
        for t in ids:
            if t.dtype != torch.int32 or t.dim() != 1 or t.shape != ids[0].shape or not t.is_contiguous():
                raise ValueError("requests must be int32 vectors of one length, contiguous")
        return ids[0].shape[0]

    def _temp(self, stream, entry, key, *args):
        """Temporary storage for a call that copies pages: its size asked for once, allocated each time (a graph keeps its own)."""
        if stream or self._home:  # on the default stream the allocator's own order does
            self._pointers.used(stream)
        size = self._sizes.get(key)
        if size is None:
            nbytes = ctypes.c_size_t(0)
            capi.check(entry(None, ctypes.byref(nbytes), self._ref, *args, None), key[0] + "(size)")
            if len(self._sizes) > 256:
                self._sizes.clear()
            size = self._sizes[key] = (nbytes.value,), ctypes.byref(nbytes)
        return dev.empty(self._refs, size[0], torch.uint8), size[1]

    def resize(self, sequences, lengths):
        """sequences[i] gets the length lengths[i] (int32 tensors).  Pages given up are there for the
        sequences that grow; one that grows into a page which others name too gets its own copy of it
        (requests are served in their order: if all of them grow, the last one keeps it).  Returns bool [n]: False where a request was refused (an id out of range, a sequence named
        before, a length out of range, not enough free pages), which changes nothing of the sequence."""
        n = self._requests(sequences, lengths)
        L = capi.lib()
        done = dev.empty(self._refs, (n,), torch.bool)
        with dev.current(self.device):
            stream = dev.stream(self.device)
            temp, nbytes = self._temp(stream, L.thrust_cdna4_pages_resize, ("pages_resize", n), None, None, n, None)
            rc = L.thrust_cdna4_pages_resize(temp.data_ptr(), nbytes, self._ref, sequences.data_ptr(), lengths.data_ptr(), n, done.data_ptr(), stream)
        if rc:
            capi.check(rc, "pages_resize")
        dev.wrote(self._all)
        return done

    def free(self, sequences):
        """The sequences give back all their pages and are empty.  Ids out of range are passed over."""
        n = self._requests(sequences)
        with dev.current(self.device):
            capi.check(capi.lib().thrust_cdna4_pages_free(self._ref, sequences.data_ptr(), n, None, dev.stream(self.device)), "pages_free")
        dev.wrote(self._own)

    def fork(self, parents, children, share=True):
        """Sequence children[i], which must be empty and no parent in the call, becomes a copy of
        parents[i]: with `share` it names the parent's full pages and gets a copy of the partly filled
        one, otherwise copies of all.  Returns bool [n]: False where refused (an id out of range, a child
        that is not empty, a parent or named before, not enough free pages)."""
        n = self._requests(parents, children)
        L = capi.lib()
        done = dev.empty(self._refs, (n,), torch.bool)
        with dev.current(self.device):
            stream = dev.stream(self.device)
            temp, nbytes = self._temp(stream, L.thrust_cdna4_pages_fork, ("pages_fork", n), None, None, n, 0, None)
            rc = L.thrust_cdna4_pages_fork(temp.data_ptr(), nbytes, self._ref, parents.data_ptr(), children.data_ptr(), n, bool(share),
                                           done.data_ptr(), stream)
        if rc:
            capi.check(rc, "pages_fork")
        dev.wrote(self._all)
        return done

    def compact(self, tables=None, refs=None):
        """Moves pages until those in use are the lowest, and renumbers.  Returns their number, int32 [1].
        With `tables` and `refs` the new ones go there and the cache's own stay as they are: the pages
        moved from keep their contents, so work in flight with the old tables may end."""
        if (tables is None) != (refs is None):
            raise ValueError("tables and refs go together")
        if dev.need_device(tables, refs) not in (None, self.device):
            raise ValueError("tensors on another device than the cache")
        tables = self._tables if tables is None else self._array(tables, self._tables.shape, None, "tables")
        refs = self._refs if refs is None else self._array(refs, self._refs.shape, None, "refs")
        L = capi.lib()
        live = dev.empty(self._refs, (1,), torch.int32)
        with dev.current(self.device):
            stream = dev.stream(self.device)
            temp, nbytes = self._temp(stream, L.thrust_cdna4_pages_compact, ("pages_compact",), None, None, None)
            rc = L.thrust_cdna4_pages_compact(temp.data_ptr(), nbytes, self._ref, tables.data_ptr(), refs.data_ptr(), live.data_ptr(), stream)
        if rc:
            if rc == 1 and tables is not self._tables:  # hipErrorInvalidValue: what else is refused has been checked
                raise ValueError("the outputs share memory with each other or the cache's arrays, and are not the same")
            capi.check(rc, "pages_compact")
        dev.wrote((tables, refs, *self.pools))
        return live
