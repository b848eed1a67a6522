"""What the paged-batch calls and the token log probabilities refuse, on the CPU: the C ABI before it touches any GPU, with
its messages, and the Python binding's checks of tensors."""
import ctypes

import pytest
import torch

from lowbit import _native, ops

FAKE, ODD8, ODD4, ODD2 = (ctypes.c_void_p(a) for a in (4096, 4104, 4100, 4098))
F16, BF16, F32 = _native.DTYPE_F16, _native.DTYPE_BF16, _native.DTYPE_F32


def norm_rope(**k):
    a = dict(qkv=FAKE, stride=2560, dtype=F16, qw=FAKE, kw=FAKE, pos=FAKE, inv=FAKE, slots=FAKE, q=FAKE, kc=FAKE, vc=FAKE, m=3,
             hq=16, hkv=2, d=128, pages=4, page=16)
    assert set(k) <= set(a)
    a.update(k)
    return _native.lib().lowbit_norm_rope_paged(a["qkv"], a["stride"], a["dtype"], a["qw"], a["kw"], 1e-6, a["pos"], a["inv"],
                                                a["slots"], a["q"], a["kc"], a["vc"], a["m"], a["hq"], a["hkv"], a["d"],
                                                a["pages"], a["page"], 0, None)


def attend(**k):
    a = dict(q=FAKE, dtype=F16, kc=FAKE, vc=FAKE, table=FAKE, width=4, starts=FAKE, lens=FAKE, out=FAKE, t=3, b=2, hq=16, hkv=2,
             d=128, pages=4, page=16, new=3, keys=64, ws=None, size=0)
    assert set(k) <= set(a)
    a.update(k)
    return _native.lib().lowbit_attention_paged(a["q"], a["dtype"], a["kc"], a["vc"], a["table"], a["width"], a["starts"],
                                                a["lens"], a["out"], a["t"], a["b"], a["hq"], a["hkv"], a["d"], a["pages"],
                                                a["page"], a["new"], a["keys"], 1.0, a["ws"], a["size"], None)


def logprobs(**k):
    a = dict(x=FAKE, dtype=F16, stride=100, t=FAKE, lp=FAKE, ent=FAKE, tv=FAKE, ti=FAKE, m=2, v=100, top=3, ws=None, size=0)
    assert set(k) <= set(a)
    a.update(k)
    return _native.lib().lowbit_token_logprobs(a["x"], a["dtype"], a["stride"], a["t"], a["lp"], a["ent"], a["tv"], a["ti"],
                                               a["m"], a["v"], a["top"], a["ws"], a["size"], None)


PAGED = [(dict(dtype=F32), 1, "F16 or BF16"), (dict(dtype=7), 1, "F16 or BF16"), (dict(d=96), 3, "head_dim"),
         (dict(hkv=3), 3, "dividing"), (dict(hkv=0), 3, "positive"), (dict(page=24), 3, "power of two"),
         (dict(page=8), 3, "power of two"), (dict(page=1 << 17), 3, "power of two"), (dict(pages=0), 3, "pages"),
         (dict(kc=ODD8), 4, "16-byte"), (dict(vc=ODD8), 4, "16-byte"), (dict(kc=None), 1, "null"), (dict(vc=None), 1, "null")]


@pytest.mark.parametrize("call,change,code,text", [(norm_rope, *c) for c in PAGED] + [(attend, *c) for c in PAGED] + [
    (norm_rope, dict(qkv=None), 1, "null"), (norm_rope, dict(pos=None), 1, "null"), (norm_rope, dict(slots=None), 1, "null"),
    (norm_rope, dict(inv=None), 1, "null"), (norm_rope, dict(q=None), 1, "null"), (norm_rope, dict(kw=None), 1, "goes with"),
    (norm_rope, dict(m=0), 3, "M must be"), (norm_rope, dict(m=1 << 31), 3, "M must be"),
    (norm_rope, dict(stride=2552), 3, "rows of qkv"), (norm_rope, dict(stride=2564), 3, "rows of qkv"),
    (norm_rope, dict(qkv=ODD8), 4, "16-byte"), (norm_rope, dict(q=ODD8), 4, "16-byte"), (norm_rope, dict(qw=ODD8), 4, "16-byte"),
    (norm_rope, dict(pos=ODD4), 4, "naturally"), (norm_rope, dict(slots=ODD4), 4, "naturally"),
    (norm_rope, dict(inv=ODD2), 4, "naturally"),
    (attend, dict(q=None), 1, "null"), (attend, dict(table=None), 1, "null"), (attend, dict(starts=None), 1, "null"),
    (attend, dict(lens=None), 1, "null"), (attend, dict(out=None), 1, "null"), (attend, dict(t=0), 3, "T, B"),
    (attend, dict(b=0), 3, "T, B"), (attend, dict(width=0), 3, "T, B"), (attend, dict(width=1 << 28), 3, "T, B"),
    (attend, dict(t=1 << 28), 3, "T, B"), (attend, dict(new=0), 3, "max_new"), (attend, dict(keys=0), 3, "max_keys"),
    (attend, dict(q=ODD8), 4, "16-byte"), (attend, dict(out=ODD8), 4, "16-byte"), (attend, dict(table=ODD2), 4, "naturally"),
    (attend, dict(lens=ODD2), 4, "naturally"), (attend, dict(starts=ODD2), 4, "naturally"),
    (attend, dict(ws=ODD8, size=1 << 20), 1, "workspace"),
    (logprobs, dict(x=None), 1, "null"), (logprobs, dict(t=None), 1, "null"), (logprobs, dict(lp=None), 1, "null"),
    (logprobs, dict(ent=None), 1, "null"), (logprobs, dict(tv=None), 1, "null"), (logprobs, dict(ti=None), 1, "null"),
    (logprobs, dict(dtype=3), 1, "dtype"), (logprobs, dict(m=0), 3, "M and V"), (logprobs, dict(v=0), 3, "M and V"),
    (logprobs, dict(v=(1 << 31) - 5), 3, "M and V"), (logprobs, dict(stride=-1), 3, "stride"),
    (logprobs, dict(m=(1 << 22) + 1), 3, "2^22"), (attend, dict(b=1 << 22), 3, "2^22"), (norm_rope, dict(m=1 << 21), 3, "2^25"),
    (logprobs, dict(top=33), 3, "top must"), (logprobs, dict(top=-1), 3, "top must"), (logprobs, dict(v=2), 3, "top must"),
    (logprobs, dict(x=ctypes.c_void_p(4097)), 4, "naturally"), (logprobs, dict(x=ODD2, dtype=F32), 4, "naturally"),
    (logprobs, dict(t=ODD4), 4, "naturally"), (logprobs, dict(ti=ODD4), 4, "naturally"), (logprobs, dict(tv=ODD2), 4, "naturally"),
    (logprobs, dict(ws=ODD8, size=1 << 20), 1, "workspace")])
def test_refused_before_any_gpu_call(call, change, code, text):
    assert call(**change) == code
    assert text in _native.lib().lowbit_last_error().decode()


def test_tensors_off_the_gpu_are_refused():
    ext, half = ops.ext(), torch.float16
    i32, i64 = (lambda *s: torch.zeros(s, dtype=torch.int32)), (lambda *s: torch.zeros(s, dtype=torch.int64))
    cache = torch.zeros(4, 2, 16, 128, dtype=half)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.norm_rope_paged(torch.zeros(3, 2560, dtype=half), None, None, 1e-6, i64(3), torch.zeros(64), i64(3),
                            torch.zeros(3, 16, 128, dtype=half), cache, cache, 16, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.attention_paged(torch.zeros(3, 16, 128, dtype=half), cache, cache, i32(2, 4), i32(3), i32(2),
                            torch.zeros(3, 16, 128, dtype=half), 3, 64, 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.token_logprobs(torch.zeros(3, 100, dtype=half), i64(3))
