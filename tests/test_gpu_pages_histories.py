"""Sequences resized past what one launch takes, in every kind of cache: tables as whole rows, counts, and every byte of the pools."""
import pytest
import torch
from test_gpu_pages import KINDS, Account, filled, ints

import risaattention_b200 as risa
from risaattention_b200 import _backend

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_status():
    yield
    torch.cuda.synchronize()
    _backend._C.device_status()


def head_rows(cache):
    """What each token of each page and head holds, as views: keys, values, and of codes their scales."""
    out = [x.view(torch.uint8) for x in (cache.keys, cache.values)]
    for scales in (cache.key_scales, cache.value_scales):
        if cache.keys.dtype == torch.int8:
            out.append(scales.view(torch.uint8).unflatten(-1, (cache.page_size, 4)))
        elif cache.keys.dtype == torch.uint8:
            out += [scales[..., :cache.page_size, None], scales[..., cache.page_size:].unflatten(-1, (cache.page_size, -1))]
    return out


class History:
    """A cache and an account of it; every call is compared with the account, bytes included."""

    def __init__(self, cache, width, batch):
        self.cache, self.width = cache, width
        pages = cache.keys.shape[0]
        self.account = Account(pages, cache.page_size, width)
        self.references = ints([0] * pages)
        self.rows, self.lengths = [[-1] * width for _ in range(batch)], [0] * batch
        self.table, self.device_lengths = ints(self.rows), ints(self.lengths)

    def resize(self, wanted):
        self.account.copies = []
        want = [x.clone() for x in head_rows(self.cache)]
        self.lengths = self.account.resize(self.rows, self.lengths, wanted)
        self.device_lengths = risa.resize_sequences(self.cache, self.references, self.table, self.device_lengths, ints(wanted))
        assert self.device_lengths.tolist() == self.lengths and self.references.tolist() == self.account.references
        assert self.table.tolist() == self.rows  # what was given back, and what lies behind a length, included
        was = [x.clone() for x in want]
        for source, to, n in self.account.copies:
            for x, old in zip(want, was):
                x[to, :, :n] = old[source, :, :n]
        assert all(torch.equal(x, y) for x, y in zip(head_rows(self.cache), want))
        return len(self.account.copies)

    def fork(self, parents):
        self.rows, self.lengths = self.account.fork(self.rows, self.lengths, parents)
        self.table, self.device_lengths = risa.fork_sequences(self.cache, self.references, self.table, self.device_lengths, ints(parents))
        assert self.table.tolist() == self.rows and self.device_lengths.tolist() == self.lengths
        assert self.references.tolist() == self.account.references


# 2 * batch * kv_heads * page * bytes of a row are 4.5 MB at least, of 4-bit rows too; one, three and eight heads, so that shares of a page are odd.
SHAPES = [(8, 128, 256, 18), (3, 64, 128, 200), (1, 16, 64, 4700), (40, 32, 64, 60)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,page,d,children", SHAPES)
def test_much_to_copy(kind, heads, page, d, children):
    assert 2 * children * heads * page * d // 2 > 4 << 20
    parents, width = max(2, children // 9), 4
    pages = 2 * children + 2 * parents + 7
    history = History(filled(pages, heads, page, d, kind), width, parents)
    g = torch.Generator().manual_seed(children)

    def lengths(low, high, n):
        return torch.randint(low, high, (n,), generator=g).tolist()
    history.resize(lengths(1, 2 * page, parents))
    history.fork([int(x) for x in torch.randint(-1, parents, (children,), generator=g)])
    shared = sum(n % page != 0 for n in history.lengths)
    assert history.resize([n + 1 if n else 0 for n in history.lengths]) == shared > children // 2
    history.resize([max(0, n - x) if i % 3 else n + x for i, (n, x) in enumerate(zip(history.lengths, lengths(0, page + 2, children)))])
    history.fork([i - i % 4 for i in range(children)])
    wanted = lengths(page, width * page + 9, children)
    assert history.resize(wanted) > children // 9                                       # some grow, some shrink,
    assert any(n < min(m, width * page) for n, m in zip(history.lengths, wanted))       # and pages run out
    history.resize([0] * children)
    assert not bool(history.references[:pages].gt(children).any())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch", [1, 7, 31, 32, 33, 100, 129, 256, 257, 600])
def test_little_to_copy(kind, batch):
    """Histories of one launch, where a sequence has several warps or one, and of more sequences than it has warps."""
    page, width = 16, 3
    pages = 3 * batch + 5
    history = History(filled(pages, 1, page, 64, kind), width, batch)
    g = torch.Generator().manual_seed(batch)

    def lengths(low, high):
        return torch.randint(low, high, (batch,), generator=g).tolist()
    history.resize(lengths(1, 2 * page))
    history.fork([i // 2 for i in range(batch)])
    history.resize([n + 1 for n in history.lengths])
    history.resize(lengths(0, width * page + 9))
    history.fork([batch - 1 - i // 3 for i in range(batch)])
    history.resize(lengths(0, width * page + 9))
    history.resize([0] * batch)
