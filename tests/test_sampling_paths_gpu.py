"""m3_sample where its ways of deciding a row meet: rows without any cut, settings
that are not numbers, borders in large vocabularies."""

import pytest
import torch

from test_sampling_gpu import T, _check

pytestmark = pytest.mark.gpu


def _overwrite_shared_memory():
    """Products whose tiles fill the SMs' shared memory with other bits."""
    for dtype in (torch.float32, torch.bfloat16):
        a = torch.full((2048, 2048), 1e30, device="cuda", dtype=dtype)
        a @ a


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(24, 257), (24, 1000), (600, 300), (4, 8192), (3, 40000)])
def test_sample_without_cuts_sets_up_its_own_tables(rows, V, dtype):
    """The default settings: no cut stands between the row's maximum and the draw,
    and nothing that an earlier kernel left in shared memory takes part."""
    g = torch.Generator().manual_seed(V + rows)
    logits = (torch.randn(rows, V, generator=g) * 2.5).to(T[dtype])
    for kw in (dict(), dict(T_=0.7), dict(k=V + 5)):
        _overwrite_shared_memory()
        _check(logits, torch.rand(rows, generator=g), **kw)
