"""CPU: the calls of test_gpu_product_paths.py reach every kernel of the dense products, each tile shape with both loaders.

``dgcn_product_path`` chooses as a launch does; a change of the sizes it chooses by shows here as a kernel that nothing tests."""
import re
import shutil
import subprocess

import pytest

from distgcn_amd import _lib
from test_gpu_product_paths import F32, HALF, INT8, PADS

AT = 1 << 20  # an aligned address: looked at, not read
TYPES = {"float32": _lib.F32, "bfloat16": _lib.BF16, "float16": _lib.F16}
# path number -> rows, columns, wave rows, wave columns, buffers where rows are loaded straight to LDS
TILES = {0: (64, 64, 2, 2, 2), 1: (128, 128, 2, 4, 2), 2: (128, 256, 2, 4, 3), 3: (192, 256, 2, 4, 2), 4: (256, 256, 2, 4, 2), 5: (128, 16, 4, 1, 2), 6: (128, 32, 4, 1, 2),
         7: (32, 64, 1, 4, 2)}
FEW = {8: (2, 4), 9: (1, 8), 10: (1, 4)}
KIND = {"int8": 0, "bfloat16": 1, "float16": 2, "float32": 3, "precise": 4}
OUT = {"float32": "float", "bfloat16": "__bf16", "float16": "_Float16"}


def _path(kind, rows, cin, ctot, groups, out, pad=0):
    lib = _lib.load()
    dtype = _lib.I8 if kind == "int8" else _lib.F32 if kind == "precise" else TYPES[kind]
    return lib.dgcn_product_path(dtype, int(kind == "precise"), AT, cin + pad, rows, cin, groups, AT, ctot, AT, TYPES[out], ctot + pad)


def _kernel(kind, path, out):
    """The kernel's name as it is compiled."""
    k, p, direct = KIND[kind], path & 15, bool(path & 16)
    if p in TILES:
        bm, bn, wm, wn, nbuf = TILES[p]
        return "k_product<%d, %d, %d, %d, %d, %d, %s>" % (k, bm, bn, wm, wn, nbuf if direct else 2, "true" if direct else "false")
    if p in FEW:
        return "k_product_few<%d, %d, %d>" % ((k,) + FEW[p])
    return "k_product_rows<%d, %s, %d, 2>" % (k, OUT[out], p - 10)


def _calls():
    """(kind, output type, sizes.., padding) of every call the GPU tests make."""
    for case in INT8:
        for pad, _ in PADS:
            for out in TYPES:
                yield ("int8", out) + case + (pad,)
    for case in HALF:
        for kind in ("bfloat16", "float16"):
            for pad, _ in PADS:
                yield (kind, kind) + case + (pad,)
    for case in F32:
        for kind in ("float32", "precise"):
            for pad in (0, 16, 3):
                yield (kind, "float32") + case + (pad,)


def _reached():
    seen = {}
    for kind, out, rows, cin, ctot, groups, pad in _calls():
        p = _path(kind, rows, cin, ctot, groups, out, pad)
        assert p >= 0
        seen.setdefault(_kernel(kind, p, out), set()).add((out, groups > 0, pad))
    return seen


def test_every_kernel_is_reached_by_a_test():
    seen = _reached()
    want = set()
    for kind in ("int8", "bfloat16", "float16"):
        want |= {_kernel(kind, p | d, "float32") for p in range(5) for d in (0, 16) if (p, d) != (4, 0)}  # (256 x 256 has no loader through registers)
        want |= {_kernel(kind, p, out) for p in (11, 12) for out in (TYPES if kind == "int8" else [kind])}
        want.add(_kernel(kind, 8, "float32"))
    want |= {_kernel("int8", p, "float32") for p in (9, 10)}
    want |= {_kernel("float32", p | d, "float32") for p in (0, 1, 5, 6, 7) for d in (0, 16)} | {_kernel("float32", p, "float32") for p in (11, 12)}
    want |= {_kernel("precise", d, "float32") for d in (0, 16)}
    assert want - set(seen) == set() and set(seen) - want == set()
    for name, how in seen.items():
        if name.startswith("k_product<0,"):  # one kernel for the three output types
            assert {out for out, _, _ in how} == set(TYPES), name


@pytest.mark.skipif(shutil.which("nm") is None, reason="no nm")
def test_no_kernel_is_compiled_that_no_call_reaches():
    symbols = subprocess.run(["nm", "-D", "--defined-only", _lib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    word = {"f": "float", "DF16b": "__bf16", "DF16_": "_Float16", "Lb0E": "false", "Lb1E": "true"}
    compiled = set()
    for name, args in re.findall(r"_ZN4dgcn\d+(k_product(?:_few|_rows)?)I((?:Li\d+E|Lb[01]E|DF16[b_]|f)+)EEv", symbols):
        compiled.add("%s<%s>" % (name, ", ".join(word.get(x) or x[2:-1] for x in re.findall(r"Li\d+E|Lb[01]E|DF16[b_]|f", args))))
    assert compiled and compiled - set(_reached()) == set() and set(_reached()) - compiled == set()


@pytest.mark.parametrize("kind", ["int8", "bfloat16", "float16"])
def test_a_call_of_few_tiles_costs_one_at_least(kind):
    """Up to five tiles of the largest shapes used to cost nothing, and the first free one won."""
    for rows, cin, ctot, groups in [(1, 64, 64, 1), (16, 64, 64, 8), (100, 128, 200, 3), (154, 32, 64, 4), (130, 64, 128, 1), (100, 256, 200, 5)]:
        assert _path(kind, rows, cin, ctot, groups, "float32" if kind == "int8" else kind) == 16
    assert _path("int8", 100, 4096, 200, 0, "float32") == 16


def test_small_outputs_stay_in_the_caches():
    streams = lambda kind, rows, cin, ctot, groups: _path(kind, rows, cin, ctot, groups, "float32") & 32
    assert not streams("int8", 154, 16, 64, 0) and streams("int8", 100000, 128, 256, 0)
    for rows, want in ((154, 0), (1000, 0), (4000, 0), (15000, 0), (20000, 32), (100000, 32)):
        assert streams("float32", rows, 32, 64, 10) == want, rows


@pytest.mark.parametrize("kw,text", [(dict(dtype=9), "unknown dtype"), (dict(dtype=_lib.I8, precise=1), "no such"), (dict(rows=0), "no such"), (dict(out=_lib.F16), "no such"),
                                     (dict(groups=0), "no such"), (dict(dtype=_lib.BF16, out=_lib.BF16, H=None), "no such"), (dict(ldh=3), "bad sizes"),
                                     (dict(cin=0), "bad sizes"), (dict(rows=2 ** 31 - 1), "more than")])
def test_path_refusals(kw, text):
    lib = _lib.load()
    ok = dict(dtype=_lib.F32, precise=0, H=AT, ldh=64, rows=5, cin=64, groups=2, W=AT, ctot=8, Y=AT, out=_lib.F32, ldy=8)
    assert lib.dgcn_product_path(*ok.values()) >= 0
    assert lib.dgcn_product_path(*{**ok, **kw}.values()) < 0 and text in lib.dgcn_last_error().decode()
