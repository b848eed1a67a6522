"""Keys that are NaN over whole parts of a split sequence: the rows that attend them are NaN, split or not."""
import pytest
import torch

import test_gpu_paged as paged
from lowbit import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("lens", [[(1, 4000)], [(1, 40000), (1, 300)], [(3, 4000)], [(150, 6000)], [(20, 4000), (1, 900)]])
def test_parts_of_nan_keys_are_not_left_out(cuda, lens, hq, hkv, d, dt):
    x = paged.batch(lens, hq, hkv, d, 32, dt, 3)
    new, keys = lens[0]
    args = (max(n for n, _ in lens), max(k for _, k in lens), d ** -0.5)
    clean = torch.empty_like(x[0])
    ops.ext().attention_paged(*x[:6], clean, *args)
    for lo, hi in ((512, 1536), (0, 1024), (0, keys - new), (keys - new - 1024, keys - new)):
        j = torch.arange(lo, hi, device="cuda")
        kc = x[1].clone()
        kc[x[3][0].long()[j // 32], 0, j % 32] = float("nan")      # of the first KV head
        for split in (True, False):
            out = torch.empty_like(clean)
            ops.ext().attention_paged(x[0], kc, *x[2:6], out, *args, split)
            g = hq // hkv
            assert bool(out[:new, :g].isnan().all()), (lo, hi, split)
            if split:
                out[:new, :g] = clean[:new, :g]
                assert torch.equal(out, clean), (lo, hi)
