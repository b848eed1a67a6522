"""Each refusal of attention_paged and attention_paged_tree, which share their checks, names the call that was made (CPU: the C ABI
before it touches any GPU)."""
import ctypes

import pytest

from lowbit import _native

FAKE, ODD8, ODD2 = (ctypes.c_void_p(a) for a in (4096, 4104, 4098))
DEFAULTS = dict(q=FAKE, dtype=_native.DTYPE_F16, kc=FAKE, vc=FAKE, table=FAKE, width=4, starts=FAKE, lens=FAKE, masks=FAKE, words=1,
                out=FAKE, t=3, b=2, hq=16, hkv=2, d=128, pages=4, page=16, new=3, keys=64, scale=1.0, ws=None, size=0)
SIZES = "t b hq hkv d width page new keys"


def run(name, **change):
    a = {**DEFAULTS, **change}
    order = "q dtype kc vc table width starts lens masks words out t b hq hkv d pages page new keys scale ws size".split()
    if name == "attention_paged":
        order = [x for x in order if x not in ("masks", "words")]
    rc = getattr(_native.lib(), f"lowbit_{name}")(*[a[x] for x in order], None)
    return rc, _native.lib().lowbit_last_error().decode()


@pytest.mark.parametrize("name", ["attention_paged", "attention_paged_tree"])
@pytest.mark.parametrize("change", [
    dict(dtype=_native.DTYPE_F32), dict(d=96), dict(hkv=3), dict(hq=65537, hkv=1), dict(page=24), dict(pages=0), dict(t=0), dict(b=0),
    dict(b=65537), dict(width=0), dict(width=1 << 27), dict(new=0), dict(keys=0), dict(q=ODD8), dict(kc=ODD8), dict(out=ODD8),
    dict(table=ODD2), dict(starts=ODD2), dict(lens=ODD2), dict(ws=ODD8, size=1 << 20)])
def test_the_call_is_named(name, change):
    rc, text = run(name, **change)
    assert rc != 0 and text.split()[0].rstrip(":") == name


@pytest.mark.parametrize("name", ["attention_paged", "attention_paged_tree"])
def test_the_workspace_query_names_the_call(name):
    for change in (dict(d=96), dict(b=0), dict(new=0)):
        a = {**DEFAULTS, **change}
        assert getattr(_native.lib(), f"lowbit_{name}_workspace")(*[a[x] for x in SIZES.split()]) == 0
        assert _native.lib().lowbit_last_error().decode().split()[0].rstrip(":") == name
