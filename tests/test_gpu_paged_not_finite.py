"""Infinities and NaN in single keys, in whole pages of keys and behind a tile's last row: attention_paged keeps them to the
rows that attend them, and keeps them there however the keys are split. Where many query heads share a KV head, all rows of a
wave, or of a tile, are one token's."""
import pytest
import torch

import test_gpu_paged as paged
from lowbit import ops

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(32, 1, 128), (40, 1, 64), (64, 1, 64), (71, 1, 128), (64, 2, 128), (128, 1, 128)])
def test_a_later_token_of_many_heads_reaches_no_earlier_one(cuda, hq, hkv, d, dt):
    """Every key of a block in turn, under bounds that choose the tiles of 32 (four waves), 64 and 128 rows."""
    new, past = 45, 20
    lens = [(new, new + past)]
    x = paged.widened(paged.batch(lens, hq, hkv, d, 16, dt, hq), 1 << 16)
    for max_new, max_keys in ((1, 600), (new, 600), (new, 60000)):
        for which, bad in ((2, NAN), (2, INF), (1, NAN)):
            clean = torch.empty_like(x[0])
            ops.ext().attention_paged(*x[:6], clean, max_new, max_keys, d ** -0.5)
            assert bool(clean.isfinite().all())
            for at in range(past - 3, past + new):
                cache = x[which].clone()
                cache[x[3][0, at // 16], 0, at % 16, 5] = bad
                out = torch.empty_like(clean)
                ops.ext().attention_paged(x[0], *(cache if i == which else x[i] for i in (1, 2)), *x[3:6], out, max_new, max_keys,
                                          d ** -0.5)
                first, g = max(0, at - past), hq // hkv
                hit = out[first:, :g, 5] if which == 2 else out[first:, :g]
                assert bool(hit.isnan().all() if bad != bad else (hit == bad).all()), (max_new, max_keys, which, bad, at)
                hit.zero_()
                want = clean.clone()
                (want[first:, :g, 5] if which == 2 else want[first:, :g]).zero_()
                assert torch.equal(out, want), (max_new, max_keys, which, bad, at)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(32, 1, 128), (64, 1, 64)])
def test_a_later_token_in_a_batch_of_single_waves(cuda, hq, hkv, d, dt):
    """Tiles of one wave, which large batches take: 2 to 5 tokens a sequence, the last with a NaN value."""
    lens = [(2 + i % 4, 2 + i % 4 + i % 50) for i in range(150)]
    x = list(paged.batch(lens, hq, hkv, d, 16, dt, 1))
    args = (1, 100, d ** -0.5)
    clean, out = torch.empty_like(x[0]), torch.empty_like(x[0])
    ops.ext().attention_paged(*x[:6], clean, *args)
    x[2] = x[2].clone()
    for b, (new, keys) in enumerate(lens):
        x[2][x[3][b, (keys - 1) // 16], :, (keys - 1) % 16, 9] = NAN
    ops.ext().attention_paged(*x[:6], out, *args)
    last = torch.tensor(x[7][1:], device="cuda") - 1
    assert bool(out[last, :, 9].isnan().all())
    out[last, :, 9] = clean[last, :, 9]
    assert torch.equal(out, clean)
