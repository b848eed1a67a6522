"""What plan_paged, attention_paged_tree, accept_drafts and beam_select refuse, on the CPU: the C ABI before it touches any GPU, with
its messages, and the Python binding's checks of tensors."""
import ctypes

import pytest
import torch

from lowbit import _native, ops

FAKE, ODD8, ODD4, ODD2, ODD1 = (ctypes.c_void_p(a) for a in (4096, 4104, 4100, 4098, 4097))
OTHER = ctypes.c_void_p(8192)
F16, F32 = _native.DTYPE_F16, _native.DTYPE_F32


def call(name, defaults, order):
    def run(**k):
        assert set(k) <= set(defaults), k
        a = {**defaults, **k}
        return getattr(_native.lib(), name)(*[a[x] for x in order.split()], None)
    return run


plan = call("lowbit_plan_paged", dict(
    table=FAKE, R=3, width=4, past=FAKE, new=FAKE, rows=None, B=3, T=9, pages=12, ps=16, parents=None, words=1, out=OTHER, starts=FAKE,
    lens=FAKE, pos=FAKE, slots=FAKE, masks=FAKE, copies=FAKE, missing=FAKE, k=None, v=None, layers=2, hkv=2, row=256, ws=None, size=0),
    "table R width past new rows B T pages ps parents words out starts lens pos slots masks copies missing k v layers hkv row ws size")
tree = call("lowbit_attention_paged_tree", dict(
    q=FAKE, dtype=F16, kc=FAKE, vc=FAKE, table=FAKE, width=4, starts=FAKE, lens=FAKE, masks=FAKE, words=1, out=FAKE, t=3, b=2, hq=16,
    hkv=2, d=128, pages=4, page=16, new=3, keys=64, scale=1.0, ws=None, size=0),
    "q dtype kc vc table width starts lens masks words out t b hq hkv d pages page new keys scale ws size")
accept = call("lowbit_accept_drafts", dict(
    tokens=FAKE, picks=FAKE, parents=FAKE, starts=FAKE, lens=FAKE, table=FAKE, width=4, k=FAKE, v=FAKE, path=FAKE, counts=FAKE,
    acc=FAKE, ends=FAKE, T=9, B=3, longest=5, layers=2, pages=12, hkv=2, ps=16, row=256),
    "tokens picks parents starts lens table width k v path counts acc ends T B longest layers pages hkv ps row")
beam = call("lowbit_beam_select", dict(
    x=FAKE, dtype=F16, stride=100, scores=FAKE, fin=None, best=FAKE, par=FAKE, tok=FAKE, req=2, beams=3, v=100, n=6, pad=0, ws=FAKE,
    size=1 << 20),
    "x dtype stride scores fin best par tok req beams v n pad ws size")

LAYERS = [(dict(v=None, k=FAKE), 1, "goes with"), (dict(k=None, v=FAKE), 1, "goes with"), (dict(k=FAKE, v=FAKE, layers=0), 3, "layers"),
          (dict(k=FAKE, v=FAKE, layers=65536), 3, "layers"), (dict(k=FAKE, v=FAKE, row=24), 3, "multiple of 16"),
          (dict(k=FAKE, v=FAKE, row=0), 3, "multiple of 16"), (dict(k=FAKE, v=FAKE, row=4112), 3, "multiple of 16"),
          (dict(k=FAKE, v=FAKE, hkv=0), 3, "layers"), (dict(k=FAKE, v=FAKE, hkv=65536, ps=65536), 3, "2^34"),
          (dict(k=ODD8, v=FAKE), 4, "16-byte"), (dict(k=FAKE, v=ODD8), 4, "16-byte"), (dict(ps=24), 3, "power of two"),
          (dict(ps=8), 3, "power of two"), (dict(ps=1 << 17), 3, "power of two"), (dict(pages=0), 3, "pages"),
          (dict(pages=1 << 31), 3, "pages")]


@pytest.mark.parametrize("run,change,code,text", [(plan, *c) for c in LAYERS] + [(accept, *c) for c in LAYERS] + [
    (plan, {k: None}, 1, "null") for k in ("table", "past", "new", "out", "starts", "lens", "pos", "slots", "copies", "missing")] + [
    (plan, {k: ODD2}, 4, "naturally") for k in ("table", "past", "new", "out", "starts", "lens", "copies", "missing", "parents")] + [
    (plan, dict(rows=ODD2), 4, "naturally"), (plan, dict(pos=ODD4), 4, "naturally"), (plan, dict(slots=ODD4), 4, "naturally"),
    (plan, dict(masks=ODD4, parents=FAKE), 4, "naturally"), (plan, dict(R=4), 3, "a row for every"),
    (plan, dict(rows=FAKE, out=FAKE), 1, "of their own"), (plan, dict(parents=FAKE, words=0), 3, "1..16 words"),
    (plan, dict(parents=FAKE, words=17), 3, "1..16 words"), (plan, dict(parents=FAKE, masks=None), 3, "1..16 words"),
    (plan, dict(B=0, R=0), 3, "R, B"), (plan, dict(B=65537, R=65537), 3, "R, B"), (plan, dict(T=-1), 3, "R, B"),
    (plan, dict(T=(1 << 28) + 1), 3, "R, B"), (plan, dict(width=0), 3, "R, B"), (plan, dict(width=(1 << 26) + 1), 3, "R, B"),
    (plan, dict(B=60000, R=60000, width=20000), 3, "R, B"), (plan, dict(B=2000, R=2000), 1, "workspace of"),
    (plan, dict(B=2000, R=2000, ws=FAKE, size=100), 1, "workspace of"),
    (plan, dict(B=2000, R=2000, ws=ODD8, size=1 << 30), 1, "workspace of"), (plan, dict(pages=1 << 20), 1, "workspace of"),
    (plan, dict(T=5000), 1, "workspace of"), (plan, dict(width=30000), 1, "workspace of"),
    (tree, dict(masks=None), 1, "null"), (tree, dict(q=None), 1, "null"), (tree, dict(out=None), 1, "null"),
    (tree, dict(words=0), 3, "1..16 words"), (tree, dict(words=17), 3, "1..16 words"), (tree, dict(masks=ODD4), 4, "naturally"),
    (tree, dict(d=96), 3, "head_dim"), (tree, dict(dtype=F32), 1, "F16 or BF16"), (tree, dict(new=0), 3, "max_new"),
    (tree, dict(t=0), 3, "T, B"), (tree, dict(ws=ODD8, size=1 << 20), 1, "workspace"), (tree, dict(page=24), 3, "power of two")] + [
    (accept, {k: None}, 1, "null") for k in ("tokens", "picks", "starts", "lens", "table", "path", "counts", "acc", "ends")] + [
    (accept, {k: ODD4}, 4, "naturally") for k in ("tokens", "picks", "acc")] + [
    (accept, {k: ODD2}, 4, "naturally") for k in ("parents", "starts", "lens", "table", "path", "counts", "ends")] + [
    (accept, dict(T=0), 3, "T, B"), (accept, dict(B=0), 3, "T, B"), (accept, dict(longest=0), 3, "T, B"),
    (accept, dict(longest=1025), 3, "T, B"), (accept, dict(width=0), 3, "T, B"), (accept, dict(B=65537), 3, "T, B")] + [
    (beam, {k: None}, 1, "null") for k in ("x", "scores", "best", "par", "tok", "ws")] + [
    (beam, dict(dtype=3), 1, "dtype"), (beam, dict(req=0), 3, "beams 1..64"), (beam, dict(beams=0), 3, "beams 1..64"),
    (beam, dict(beams=65), 3, "beams 1..64"), (beam, dict(req=1 << 22), 3, "2^22"), (beam, dict(v=0), 3, "V must"),
    (beam, dict(v=(1 << 31) - 5), 3, "V must"), (beam, dict(stride=-1), 3, "stride"), (beam, dict(n=0), 3, "n must"),
    (beam, dict(n=33), 3, "n must"), (beam, dict(v=1, n=4), 3, "n must"), (beam, dict(fin=FAKE, pad=-1), 1, "pad"),
    (beam, dict(fin=FAKE, pad=100), 1, "pad"), (beam, dict(x=ODD1), 4, "naturally"), (beam, dict(x=ODD2, dtype=F32), 4, "naturally"),
    (beam, dict(scores=ODD2), 4, "naturally"), (beam, dict(par=ODD4), 4, "naturally"), (beam, dict(tok=ODD4), 4, "naturally"),
    (beam, dict(ws=ODD8), 1, "workspace"), (beam, dict(size=6 * 64 - 1), 1, "workspace")])
def test_refused_before_any_gpu_call(run, change, code, text):
    assert run(**change) == code
    assert text in _native.lib().lowbit_last_error().decode()


def test_workspace_of_a_plan():
    """None for what one workgroup plans, enough beyond, nothing for sizes that are refused."""
    size = _native.lib().lowbit_plan_paged_workspace
    assert size(8, 200, 900, 3000, 16) == 0
    assert size(256, 2000, 900, 300000, 16) > 2 * 300000 // 8
    assert size(0, 2000, 900, 300000, 16) == 0 and size(8, 200, 900, 3000, 24) == 0


def test_tensors_off_the_gpu_are_refused():
    ext, half = ops.ext(), torch.float16
    i32, i64 = (lambda *s: torch.zeros(s, dtype=torch.int32)), (lambda *s: torch.zeros(s, dtype=torch.int64))
    cache = torch.zeros(4, 2, 16, 128, dtype=half)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.plan_paged(i32(3, 4), i32(3), i32(3), 9, 12, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.attention_paged_tree(torch.zeros(3, 16, 128, dtype=half), cache, cache, i32(2, 4), i32(3), i32(2), i64(3, 1),
                                 torch.zeros(3, 16, 128, dtype=half), 3, 64, 1.0)
    with pytest.raises(RuntimeError, match="words"):
        ext.attention_paged_tree(torch.zeros(3, 16, 128, dtype=half), cache, cache, i32(2, 4), i32(3), i32(2), i64(3, 17),
                                 torch.zeros(3, 16, 128, dtype=half), 3, 64, 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.accept_drafts(i64(9), i64(9), i32(9), i32(4), i32(3), i32(3, 4), (cache, cache), 5)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.beam_select(torch.zeros(6, 100, dtype=half), torch.zeros(2, 3), 6)
