"""attention_paged where scores are so large that 32 bits hold them to whole numbers or less. Only one dim of q and k differs
from zero and its values have few bits, so that every score is exact in 32 bits, equal ones are equal, and the others lie so far
below that their weight is zero: the output is the mean of the largest scores' values, to the bound of test_gpu_paged.py without
its term for scores."""
import pytest
import torch

import test_gpu_paged as paged
from lowbit import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("lens", [[(1, 40)], [(1, 5000)], [(40, 700)], [(200, 2500), (1, 300)]])
def test_large_scores(cuda, lens, hq, hkv, d, dt):
    g = torch.Generator(device="cuda").manual_seed(5)
    for size, scale in ((1000.0, 0.09), (9000.0, 0.09), (30000.0, 0.125), (50000.0, 0.3), (60000.0, 2.0), (60000.0, -2.0),
                        *(((1e15, 0.1), (1e18, -1.0)) if dt is torch.bfloat16 else ())):
        x = list(paged.batch(lens, hq, hkv, d, 32, dt, 2))
        q = torch.zeros_like(x[0])
        q[..., 3] = (size * (0.5 + 0.5 * torch.rand(q.shape[:2], generator=g, device="cuda"))).to(dt)
        out = torch.empty_like(q)
        for b, (new, keys) in enumerate(lens):
            k = torch.zeros_like(x[6][b][0])
            # a few largest in the past and the others 1/8 or more below; the first key is one of the largest, so that every
            # row attends one
            k[..., 3] = (size / 2 * torch.rand(k.shape[:2], generator=g, device="cuda")).to(dt)
            top = torch.rand(k.shape[:2], generator=g, device="cuda") < 0.01
            top[0] = True
            k[..., 3][top] = size
            if scale < 0:
                k = -k
            j = torch.arange(keys, device="cuda")
            x[1][x[3][b].long()[j // 32], :, j % 32] = k
            x[6][b] = (k, x[6][b][1])
        ops.ext().attention_paged(q, *x[1:6], out, max(n for n, _ in lens), max(k for _, k in lens), scale)
        for b, (new, keys) in enumerate(lens):
            k, v = x[6][b]
            last = keys - new + torch.arange(new, device="cuda")
            for h in range(hkv):
                size_of = k[:, h, 3].double().abs()
                p = ((size_of == size_of.max())[None, :] & (torch.arange(keys, device="cuda")[None, :] <= last[:, None])).double()
                p /= p.sum(-1, keepdim=True)
                want, room = (p @ v[:, h].double())[:, None], (p @ v[:, h].double().abs())[:, None]
                tol = room * (paged.half_step(dt) + (keys / 16 + 64) * paged.U) + paged.half_step(dt) * want.abs() + paged.least(dt)
                got = out[x[7][b]:x[7][b + 1], h * (hq // hkv):(h + 1) * (hq // hkv)].double()
                assert bool(((got - want).abs() <= tol).all()), (size, scale, b, h, got.isfinite().all())


def test_a_scale_that_is_not_a_number_is_not_hidden(cuda):
    for lens in ([(1, 40)], [(1, 5000)], [(200, 700)]):
        x = paged.batch(lens, 16, 2, 128, 32, torch.float16, 2)
        out = torch.zeros_like(x[0])
        ops.ext().attention_paged(*x[:6], out, max(n for n, _ in lens), max(k for _, k in lens), float("nan"))
        assert bool(out.isnan().all()), lens
