"""NaN at the shard's first id and rows of only NaN, in lists that hold empty places: the
largest possible entry and none beside it, where lists merge."""

from __future__ import annotations

import pytest
import torch

import test_top_gpu as top

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def _rows(v, dtype, g):
    x = (torch.randn(6, v, generator=g) * 3).to(dtype)
    x[0, 0] = NAN
    x[1] = NAN
    x[2, 0], x[2, v - 1] = NAN, INF
    x[3, ::3] = NAN
    x[4] = -INF
    x[4, 0] = NAN
    return x


# A last slab narrower than k (v = 3 4096 + 50 is cut to four), lists of up to 1024 entries
# together and of more, one slab alone.
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("v,k", [(3 * 4096 + 50, 200), (3 * 4096 + 50, 256), (2 * 4096 + 1, 300),
                                 (3 * 4096 + 50, 300), (5 * 8192 + 3, 512), (2 * 4096 + 7, 45),
                                 (4097, 500), (600, 512)])
def test_nan_at_the_first_id(v, k, dtype):
    x = _rows(v, dtype, torch.Generator().manual_seed(v + k))
    top._check(x, k)
    for i in range(6):
        top._check(x[i:i + 1], k)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("tp,per,k", [(5, 150, 200), (6, 170, 170), (10, 80, 100), (3, 341, 341),
                                      (64, 15, 16), (20, 45, 51), (20, 45, 500), (70, 9, 14)])
def test_shards_narrower_than_k(tp, per, k, dtype):
    """Ranks that hold fewer columns than are wanted."""
    from nmce import _lib as L
    lib = L.load()
    v = tp * per
    x = _rows(v, dtype, torch.Generator().manual_seed(tp))
    n, code = x.shape[0], L.dtype_code(dtype)
    parts = torch.zeros(tp, n, k + 1, dtype=torch.int64, device=DEV)
    stream = L.stream_handle(torch.device(DEV))
    for r in range(tp):
        mine = x[:, r * per:(r + 1) * per].contiguous().to(DEV)
        ws = torch.empty(lib.nmce_top_workspace_bytes(n, per, k), dtype=torch.uint8, device=DEV)
        L.check(lib.nmce_top_logits(mine.data_ptr(), code, n, per, per, r * per, k, 1.0,
                                    parts[r].data_ptr(), None, None, None, ws.data_ptr(),
                                    ws.numel(), stream), "top")
    values = torch.empty(n, k, dtype=dtype, device=DEV)
    ids = torch.empty(n, k, dtype=torch.int64, device=DEV)
    norm = torch.empty(n, device=DEV)
    L.check(lib.nmce_top_merge(parts.data_ptr(), tp, code, n, k, 1.0, values.data_ptr(),
                               ids.data_ptr(), norm.data_ptr(), stream), "merge")
    want = torch.sort(x, dim=-1, descending=True, stable=True)
    assert torch.equal(ids.cpu(), want.indices[:, :k])
    got, held = values.cpu(), want.values[:, :k]
    assert torch.equal(torch.isnan(got), torch.isnan(held))
    assert torch.equal(got.nan_to_num(7.0), held.nan_to_num(7.0))
    assert torch.equal(torch.isnan(norm.cpu()), torch.isnan(x).any(1))
