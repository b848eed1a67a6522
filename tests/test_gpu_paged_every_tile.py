"""attention_paged where a call has more tiles of query rows than the workspace has records, or a workspace of a few records:
every row is computed, and nothing behind the workspace is written. Bounds as in test_gpu_paged.py."""
import pytest
import torch

import test_gpu_paged as paged
from lowbit import _native, ops

pytestmark = pytest.mark.gpu


def called(x, lens, workspace_bytes, scale):
    """The C entry with a workspace of so many bytes, 4 KB behind it watched."""
    q, kc, vc, table, starts, kv_lens = x[:6]
    out = torch.full_like(q, float("nan"))
    ws = torch.full((workspace_bytes + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    _native.check(ops.ext().lib.lowbit_attention_paged(
        q.data_ptr(), _native.DTYPE_F16 if q.dtype is torch.float16 else _native.DTYPE_BF16, kc.data_ptr(), vc.data_ptr(),
        table.data_ptr(), table.shape[1], starts.data_ptr(), kv_lens.data_ptr(), out.data_ptr(), q.shape[0], len(lens),
        q.shape[1], kc.shape[1], q.shape[2], kc.shape[0], kc.shape[2], max(n for n, _ in lens), max(k for _, k in lens), scale,
        ws.data_ptr(), workspace_bytes, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert bool((ws[workspace_bytes:] == 0x5A).all())
    return out


def check(out, x, lens, scale, least_row=0):
    """Every row from least_row of its sequence on against 64 bits, and no row left out."""
    assert not bool(out.isnan().any()), out.isnan().nonzero()[:3].tolist()
    for b, (new, keys) in enumerate(lens):
        if new > least_row:
            rows = slice(x[7][b] + least_row, x[7][b + 1])
            want, tol = paged.attend_want(x[0][rows], *x[6][b], new - least_row, keys, scale)
            assert bool(((out[rows].double() - want).abs() <= tol).all()), (b, new, keys)


# sequences of more than 2048 tiles of 128 query rows times KV heads
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,new,past", [(28, 4, 128, 9500, 0), (32, 8, 128, 8200, 0), (64, 8, 64, 4200, 300), (12, 12, 64, 22000, 0)])
def test_long_prompts_are_whole(cuda, hq, hkv, d, new, past, dt):
    lens = [(1, 700), (new, new + past), (3, 50)]
    x = paged.batch(lens, hq, hkv, d, 64, dt, new)
    for split in (True, False):
        out = torch.full_like(x[0], float("nan"))
        ops.ext().attention_paged(*x[:6], out, new, new + past, d ** -0.5, split)
        check(out, x, lens, d ** -0.5, new - 150)
        check(out[:1], x, lens[:1], d ** -0.5)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("records", [1, 2, 3, 8, 64, 300])
def test_small_workspaces_split_less(cuda, records, dt):
    for hq, hkv, d, lens, rows in ((28, 4, 128, [(1, 900 + 97 * i) for i in range(31)], 32),
                                   (28, 4, 128, [(1, 30000), (1, 1)], 32), (14, 2, 64, [(2, 5000), (1, 800), (3, 2000)], 32),
                                   (28, 4, 128, [(700, 700), (300, 2500), (1, 4000)], 128), (14, 2, 64, [(1500, 1500)], 128),
                                   (16, 2, 128, [(20, 1000), (9, 600)], 64)):
        x = paged.batch(lens, hq, hkv, d, 32, dt, records)
        print(hq, hkv, d, lens[:3], records, flush=True)
        out = called(x, lens, records * rows * (d + 4) * 4, d ** -0.5)
        check(out, x, lens, d ** -0.5)
        check(called(x, lens, records * rows * (d + 4) * 4 - 16, d ** -0.5), x, lens, d ** -0.5)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_more_workspace_than_asked_for_changes_nothing(cuda, dt):
    for hq, hkv, d, lens in ((28, 4, 128, [(1, 900 + 97 * i) for i in range(31)]), (28, 4, 128, [(1, 30000), (1, 1)]), (12, 1, 128, [(2, 65000)]),
                             (14, 2, 64, [(2, 5000), (1, 800), (3, 2000)]), (28, 4, 128, [(1, 1500)] * 200), (28, 4, 128, [(1, 100)] * 280 + [(1, 3000)]),
                             (28, 4, 128, [(700, 700), (300, 2500), (1, 4000)]), (14, 2, 64, [(1500, 1500)]), (16, 2, 128, [(20, 1000), (9, 600)])):
        x = paged.batch(lens, hq, hkv, d, 32, dt, len(lens))
        asked = ops.ext().lib.lowbit_attention_paged_workspace(x[0].shape[0], len(lens), hq, hkv, d, x[3].shape[1], 32,
                                                               max(n for n, _ in lens), max(k for _, k in lens))
        print(hq, hkv, d, lens[:2], asked, flush=True)
        assert asked
        one = called(x, lens, asked, d ** -0.5)
        assert torch.equal(one, called(x, lens, asked + (200 << 20), d ** -0.5))
        out = torch.full_like(one, float("nan"))
        ops.ext().attention_paged(*x[:6], out, max(n for n, _ in lens), max(k for _, k in lens), d ** -0.5)
        assert torch.equal(out, one)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hkv,d,n", [(6, 2, 64, 65536), (28, 4, 128, 5001)])
def test_as_many_sequences_as_are_taken(cuda, hq, hkv, d, n, dt):
    """One token a sequence on 1 .. 16 keys of one page; pages are shared. Bound as in test_gpu_paged.py (16 keys)."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    kc, vc = (torch.randn(50, hkv, 16, d, generator=gen, device="cuda").to(dt) for _ in range(2))
    q = torch.randn(n, hq, d, generator=gen, device="cuda").to(dt)
    page, keys = (torch.randint(0, top, (n,), generator=gen, device="cuda", dtype=torch.int32) for top in (50, 16))
    keys += 1
    out = torch.full_like(q, float("nan"))
    ops.ext().attention_paged(q, kc, vc, page[:, None].contiguous(), torch.arange(n + 1, dtype=torch.int32, device="cuda"), keys, out,
                              1, 16, d ** -0.5)
    at, dead = page.long(), torch.arange(16, device="cuda")[None, :] >= keys[:, None]
    for h in range(hq):
        k, v, x = kc[at, h // (hq // hkv)].double(), vc[at, h // (hq // hkv)].double(), q[:, h].double()
        prod = k * x[:, None]
        p = torch.softmax((prod.sum(-1) * d ** -0.5).masked_fill(dead, -float("inf")), -1)[..., None]
        want, size = (p * v).sum(1), (p * v.abs()).sum(1)
        ds = (d + 8) * paged.U * (prod.abs().sum(-1) * d ** -0.5).masked_fill(dead, 0).amax(-1, keepdim=True)
        tol = size * (paged.half_step(dt) + 2 * ds + 65 * paged.U) + paged.half_step(dt) * want.abs() + paged.least(dt)
        assert bool(((out[:, h].double() - want).abs() <= tol).all()), h
