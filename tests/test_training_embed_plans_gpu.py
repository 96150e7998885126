"""The codebook embedding's gradient beyond the smallest sizes of its sort: longer
runs and chunks, several chunks with few histograms, the most rows and entries."""

from __future__ import annotations

import pytest
import torch

import training_ref as ref
from fast_mimi_amd import training as tr

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("b,books,frames,entries,dim,dtype", [
    (1, 2, 20_000, 2048, 24, torch.float32),      # runs of 128 rows
    (7, 1, 10_001, 2048, 16, torch.bfloat16),     # 70007 rows: chunks of 8192
    (1, 1, 270_000, 300, 8, torch.float16),       # runs of 512, chunks of 32768
    (3, 2, 3001, 2049, 8, torch.float32),         # four histograms, three chunks
    (2, 1, 4501, 8193, 8, torch.bfloat16),        # one histogram
    (1, 2, 9000, 32768, 5, torch.float16),        # the most entries, single elements
    (1, 1, 70_001, 32768, 8, torch.float32),
    (32, 1, 65_535, 17, 8, torch.bfloat16),       # the most rows
])
@pytest.mark.parametrize("codes", ["uniform", "skewed", "one", "sorted"])
def test_embedding_gradient_of_many_rows(b, books, frames, entries, dim, dtype, codes):
    g = torch.Generator().manual_seed(1)
    named = torch.randint(-1, entries, (b, books, frames), generator=g)
    if codes == "skewed":
        named = torch.where(torch.rand(named.shape, generator=g) < 0.6, min(3, entries - 1), named)
    elif codes == "one":
        named = torch.full_like(named, entries - 1)
    elif codes == "sorted":  # long stretches of one code each, the last entries without any
        named = (torch.arange(frames) * min(entries, 40) // frames).expand(b, books, frames).contiguous()
    table = torch.randn(books, entries, dim, generator=g).to(dtype)
    grad = torch.randn(b, frames, dim, generator=g).to(dtype)
    want, bound = ref.embedding(named, table, grad, 0.5)
    named, table, grad = named.to(DEV), table.to(DEV), grad.to(DEV)
    got = {"out": tr.code_embedding_forward(named, table, 0.5), "dtable": tr.code_embedding_backward(grad, named, table, 0.5)}
    for n, x in got.items():
        ref.assert_within(n, x, want[n], bound[n])
    assert torch.equal(got["dtable"], tr.code_embedding_backward(grad, named, table, 0.5))
