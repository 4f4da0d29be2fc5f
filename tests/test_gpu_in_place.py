"""C entries whose output takes the place of an input of the same kind, called with the tensors' addresses."""
import ctypes

import pytest
import torch
from test_gpu_pages import Account, filled, ints
from test_serving_launches_cpu import LIBRARY

import risaattention_b200 as risa

pytestmark = pytest.mark.gpu


class Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("keys", "values", "key_scales", "value_scales")] + [(n, ctypes.c_int) for n in ("pages", "kv_heads", "page_size", "head_dim", "dtype_code")]

    def __init__(self, cache):
        code = {torch.float16: 1, torch.bfloat16: 2, torch.int8: 4, torch.uint8: 5}[cache.keys.dtype]
        super().__init__(*(None if x is None else x.data_ptr() for x in cache.tensors), *cache.keys.shape[:3], cache.head_dim, code)


class Step(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("page_table", "lengths", "query_offsets")] + [(n, ctypes.c_int) for n in ("batch", "table_width", "tokens")]


def library():
    lib = ctypes.CDLL(str(LIBRARY))
    lib.risa_b200_resize_scratch_size.restype = ctypes.c_size_t
    return lib


def at(x):
    return ctypes.c_void_p(x.data_ptr())


@pytest.mark.parametrize("granted_is", ["lengths", "new_lengths"])
@pytest.mark.parametrize("heads,page", [(1, 16), (8, 128)])  # little to copy, and much
def test_lengths_resized_in_place(granted_is, heads, page):
    lib, pages, width, batch = library(), 150, 5, 20
    cache = filled(pages, heads, page, 256, torch.uint8)
    references, account = ints([0] * pages), Account(pages, page, width)
    table, rows = ints([[-1] * width] * batch), [[-1] * width for _ in range(batch)]
    lengths, now = ints([0] * batch), [0] * batch
    g = torch.Generator().manual_seed(heads)
    c = Cache(cache)
    scratch = torch.empty(lib.risa_b200_resize_scratch_size(ctypes.byref(c), batch), dtype=torch.uint8, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for step in range(5):
        if step == 2:  # every second sequence now shares the pages of the one in front of it
            wanted = [n if s % 2 == 0 else 0 for s, n in enumerate(now)]
            now = account.resize(rows, now, wanted)
            lengths = risa.resize_sequences(cache, references, table, lengths, ints(wanted))
            parents = [s - s % 2 for s in range(1, batch, 2)]
            more, more_now = account.fork(rows, now, parents)
            device_rows, device_lengths = risa.fork_sequences(cache, references, table, lengths, ints(parents))
            rows[1::2], now[1::2] = more, more_now
            table[1::2], lengths[1::2] = device_rows, device_lengths
        account.copies = []
        wanted = torch.randint(0, 3 * page, (batch,), generator=g).tolist() if step != 2 else [n + 1 for n in now]
        device_wanted, was = ints(wanted), [x.clone() for x in cache.tensors]
        granted = lengths if granted_is == "lengths" else device_wanted
        old = lengths.clone()
        assert lib.risa_b200_resize_sequences(ctypes.byref(c), at(references), at(table), width, at(lengths), at(device_wanted), batch, at(granted), at(scratch),
                                              ctypes.c_size_t(scratch.numel()), stream) == 0
        now = account.resize(rows, now, wanted)
        assert granted.tolist() == now and references.tolist() == account.references and table.tolist() == rows
        assert granted_is == "lengths" or torch.equal(old, lengths)
        for source, to, n in account.copies:
            assert torch.equal(cache.keys[to, :, :n], was[0][source, :, :n]) and torch.equal(cache.values[to, :, :n], was[1][source, :, :n])
        lengths = granted
        assert step != 2 or len(account.copies) > 10


def test_lengths_evicted_in_place():
    """Heads whose largest weights lie behind the budget, so that a head which took the new length for the old one would keep others."""
    lib, heads, page, width, budget = library(), 64, 16, 40, 48
    batch = 30
    cache = filled(batch * (width + 3), heads, page, 64, torch.bfloat16)
    table = torch.arange(batch * width, dtype=torch.int32, device="cuda").view(batch, width)
    target = torch.arange(batch * width, batch * (width + 3), dtype=torch.int32, device="cuda").view(batch, 3)
    lengths = torch.arange(11, 11 + 20 * batch, 20, dtype=torch.int32, device="cuda")
    weights = torch.rand(batch, heads, width * page, device="cuda") + torch.arange(width * page, device="cuda")
    want = risa.evict_from_cache(cache, table, lengths, weights, target, budget=budget, recent=5)
    kept, new_weights = torch.empty_like(want.kept), torch.empty_like(want.weights)
    step = Step(table.data_ptr(), lengths.data_ptr(), None, batch, width, batch)
    assert lib.risa_b200_cache_evict(ctypes.byref(Cache(cache)), ctypes.byref(step), at(weights), at(target), 3, budget, 5, at(kept), at(lengths), at(new_weights),
                                     ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    assert torch.equal(lengths, want.lengths) and torch.equal(kept, want.kept) and torch.equal(new_weights, want.weights)


def test_a_table_compacted_in_place():
    lib, pages, heads, page, width, batch = library(), 700, 2, 16, 12, 50
    lib.risa_b200_compact_scratch_size.restype = ctypes.c_size_t
    cache, target = filled(pages, heads, page, 64, torch.int8), filled(batch * width, heads, page, 64, torch.int8, seed=2)
    references, table = ints([0] * pages), ints([[-1] * width] * batch)
    lengths = risa.resize_sequences(cache, references, table, ints([0] * batch), ints([s * 4 for s in range(batch)]))
    lengths = risa.resize_sequences(cache, references, table, lengths, ints([s * 4 if s % 3 else 0 for s in range(batch)]))
    want = risa.compact_cache(cache, references, table, lengths, target)
    here, there = Cache(cache), Cache(target)
    scratch = torch.empty(lib.risa_b200_compact_scratch_size(ctypes.byref(here), ctypes.byref(there)), dtype=torch.uint8, device="cuda")
    counts, used = torch.empty_like(want.references), torch.empty_like(want.used)
    step = Step(table.data_ptr(), lengths.data_ptr(), None, batch, width, batch)
    assert lib.risa_b200_cache_compact(ctypes.byref(here), at(references), ctypes.byref(step), ctypes.byref(there), at(table), at(counts), at(used), at(scratch),
                                       ctypes.c_size_t(scratch.numel()), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    assert torch.equal(table, want.page_table) and torch.equal(counts, want.references) and torch.equal(used, want.used)
