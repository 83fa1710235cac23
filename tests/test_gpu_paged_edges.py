"""Calls over a paged KV cache at its edges."""
import numpy as np
import pytest

from test_gpu_paged import be, floats, u32  # noqa: F401  (be: the module's backend)

pytestmark = pytest.mark.gpu


def test_more_key_blocks_than_the_line_of_work_counts(be):
    """2^31 key blocks and more (here one page under every table entry): OutOfRange, and nothing is computed for any request."""
    from ojas_b200 import DType, OjasError
    page, width = 1 << 24, 127
    places = width * page
    for kind, d, batch, heads, tokens in ((DType.F32, 32, 128, 1, 1), (DType.BF16, 32, 300, 1, 1), (DType.BF16, 64, 2, 1, 40000), (DType.BF16, 64, 3, 1, 3000)):
        pages = be.zeros((1, page, 1, d), kind)
        new = np.full(batch, tokens)
        cached = places - new - 5
        if batch == 3:
            cached[:2] = 100                                                   # others next to one request that is too long by itself
            new[2], heads = 40000, 1
            cached[2] = places - 40001
        n = int(new.sum())
        q, out = be.zeros((n, heads, d), kind), floats(be, np.full((n, heads, d), 7.0, np.float32), kind == DType.BF16)
        lse = be.upload(np.full((n, heads), 7.0, np.float32))
        be.paged_attention_forward(q, pages, pages, u32(be, np.zeros((batch, width))), u32(be, cached), u32(be, np.concatenate([[0], np.cumsum(new)])), out=out, lse=lse)
        with pytest.raises(OjasError) as e:
            be.sync()
        assert e.value.kind == "OutOfRange"
        assert np.all(out.numpy() == 7.0) and np.all(lse.numpy() == 7.0)
        del pages
