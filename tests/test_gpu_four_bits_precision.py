"""Up to 32 query rows of a key head over a cache in 4 bits: a probability times its token's scale is held with fp16's eleven bits, for bf16 queries
too."""
import four_bits_util as F
import pytest
import serving_util as U
import torch
from test_gpu_serving import BF16, F16

import risaattention_b200 as risa

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def prepared(monkeypatch):
    monkeypatch.setattr(U, "cached", F.cached)


def rounded(batch, to):
    """(outputs with every probability times scale rounded once to type ``to``, the largest such product of each row), in 64 bits."""
    q, page = batch.q.double().cpu(), batch.cache.page_size
    out, largest = torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64)
    first = 0
    for s, count in enumerate(batch.chunks):
        k, v = U.cached(batch, s).cpu(), U.cached(batch, s, "values").cpu()
        n = k.shape[1]
        ids = batch.table[s, :-(-n // page)].long()
        token = F.power(F.scales_of(batch.cache.value_scales[ids], page)[0].transpose(0, 1).flatten(1)[:, :n]).cpu()  # [kv_heads, n]
        mask, group = U.seen(n, count, True, None, "cpu"), q.shape[1] // k.shape[0]
        for h in range(q.shape[1]):
            p = (q[first:first + count, h] @ k[h // group].T * q.shape[-1] ** -0.5).masked_fill(~mask, -torch.inf).softmax(-1)
            product = p * token[h // group]
            largest[first:first + count, h] = product.amax(-1)
            unit = product.amax(-1, keepdim=True)
            out[first:first + count, h] = (product / unit).to(to).double() * unit @ (v[h // group] / token[h // group][:, None])
        first += count
    return out, largest


# Short sequences, whose few rounded products do not average out.
CASES = [
    ([2, 3, 4, 5, 6, 7, 9, 12], [1] * 8, (16, 2), 128, 16),
    ([2, 3, 4, 5, 6, 7, 9, 12], [1] * 8, (16, 1), 64, 32),
    ([2, 3, 4, 5, 6, 7, 9, 40], [1] * 8, (8, 2), 256, 64),
    ([5, 6, 12, 9], [4, 3, 8, 1], (8, 2), 128, 16),   # 32 rows of a key head
    ([5, 6, 12, 9], [4, 3, 8, 1], (4, 1), 64, 16),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_few_rows(case, dtype):
    lengths, chunks, (q_heads, kv_heads), d, page = case
    b = F.batch_of(lengths, chunks, q_heads=q_heads, kv_heads=kv_heads, head_dim=d, page=page, dtype=dtype, seed=d)
    out, _ = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=None if set(chunks) == {1} else b.offsets, return_lse=True)
    want, _, spread, size = (x.cpu() for x in U.attention(b))
    planted, largest = rounded(b, torch.bfloat16)
    # The output rounded once; scores as in assert_attention; a product rounded once to fp16, 2^-11 of it or, where it is small, 2^-25 of the row's
    # largest, times codes and group scales of at most 7 * 448.
    score = size * d * 2.0 ** -23 + 2.0 ** -20 * (1 + size)
    bound = torch.finfo(dtype).eps / 2 * want.abs() + spread * (2.0 ** -11 + 2.1 * score[..., None])
    bound += max(lengths) * 2.0 ** -25 * 3136 * largest[..., None] + torch.finfo(dtype).tiny
    error = (out.double().cpu() - want).abs()
    assert bool((error <= bound).all()), f"{float((error / bound).max()):.2f} of the bound"
    # products with bf16's eight bits would be seen
    assert bool(((planted - want).abs() > bound).any())
