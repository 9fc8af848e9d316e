"""Linear with 4-bit weights, host side: the C ABI's structure and argument
checks (no launch), and the refusal of CPU tensors."""

import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from longvideosparseattention_b200 import _native as N
from tests.conftest import ROOT

FAKE = 1 << 20  # aligned, never read


def _args(**kw):
    a = N.LvsaW4Linear(FAKE, FAKE, FAKE, None, FAKE, 64, 32, 0, 32, 64, 64, 0, 0, 0, 0, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_struct_layout():
    probe = r'''
#include <stdio.h>
#include <stddef.h>
#include "lvsa_b200.h"
int main(void){ printf("%zu %zu %zu\n", sizeof(LvsaW4Linear), offsetof(LvsaW4Linear, m), offsetof(LvsaW4Linear, activation)); return 0;}
'''
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
        with open(c, "w") as fh:
            fh.write(probe)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        got = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(N.LvsaW4Linear), N.LvsaW4Linear.m.offset, N.LvsaW4Linear.activation.offset]


def test_checks():
    lib = N.load()
    call = lambda a: lib.lvsa_w4_linear(ctypes.byref(a), None)  # noqa: E731
    assert call(_args()) == N.LVSA_OK  # no rows: nothing to launch
    assert lib.lvsa_w4_linear(None, None) == N.LVSA_ERR_INVALID_ARG
    for bad in (dict(m=-1), dict(n=0), dict(k=0), dict(tiles=None), dict(scales=None), dict(activation=2),
                dict(m=1, x=None), dict(m=1, out=None), dict(m=1, ldx=63), dict(m=1, ldo=31)):
        assert call(_args(**bad)) == N.LVSA_ERR_INVALID_ARG, bad
    for bad in (dict(group=16), dict(group=256), dict(x_dtype=2), dict(out_dtype=9), dict(bias=FAKE, bias_dtype=2),
                dict(scale_dtype=3)):
        assert call(_args(**bad)) == N.LVSA_ERR_UNSUPPORTED, bad
    for bad in (dict(tiles=FAKE + 8), dict(scales=FAKE + 4)):
        assert call(_args(**bad)) == N.LVSA_ERR_ALIGNMENT, bad
    for bad in (dict(n=2 ** 30 + 1, ldo=2 ** 31), dict(k=2 ** 30 + 1, ldx=2 ** 31), dict(m=65536)):
        assert call(_args(**bad)) == N.LVSA_ERR_UNSUPPORTED, bad
    size = ctypes.c_int64()
    for n, k in ((2 ** 30 + 1, 1), (1, 2 ** 30 + 1)):
        assert lib.lvsa_w4_bytes(n, k, ctypes.byref(size)) == N.LVSA_ERR_UNSUPPORTED
        assert lib.lvsa_w4_pack(FAKE, k, n, k, FAKE, None) == N.LVSA_ERR_UNSUPPORTED
    assert lib.lvsa_w4_bytes(17, 65, ctypes.byref(size)) == N.LVSA_OK and size.value == 2 * 2 * 512
    assert lib.lvsa_w4_bytes(0, 65, ctypes.byref(size)) == N.LVSA_ERR_INVALID_ARG
    assert lib.lvsa_w4_bytes(1, 1, None) == N.LVSA_ERR_INVALID_ARG
    assert lib.lvsa_w4_pack(None, 1, 1, 1, FAKE, None) == N.LVSA_ERR_INVALID_ARG
    assert lib.lvsa_w4_pack(FAKE, 7, 1, 8, FAKE, None) == N.LVSA_ERR_INVALID_ARG
    assert lib.lvsa_w4_pack(FAKE, 8, 1, 8, FAKE + 8, None) == N.LVSA_ERR_ALIGNMENT


def test_cpu_tensors_are_refused():
    from longvideosparseattention_b200.linear_w4 import pack_w4, quantize_w4
    with pytest.raises(RuntimeError):
        pack_w4(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.bfloat16), 64)
    with pytest.raises(RuntimeError):
        quantize_w4(torch.zeros(4, 64))


def test_quantize_refuses_what_has_no_codes():
    """An infinity or NaN anywhere, or a scale past its type: before any kernel runs."""
    from longvideosparseattention_b200.linear_w4 import quantize_w4
    for bad, dtype in ((float("inf"), torch.bfloat16), (float("-inf"), torch.float16), (float("nan"), torch.bfloat16),
                       (1e6, torch.float16)):
        weight = torch.ones(3, 100)
        weight[2, 99] = bad
        with pytest.raises(ValueError):
            quantize_w4(weight, 32, dtype)
    with pytest.raises(ValueError):
        quantize_w4(torch.full((1, 64), 1e300, dtype=torch.float64))


def test_weights_that_do_not_fit_their_sizes_are_refused():
    """The kernel goes by n, k and group: tensors of other sizes would be read out of range."""
    import dataclasses

    from longvideosparseattention_b200.linear_w4 import W4Weight
    BF = torch.bfloat16

    def make(n, k, group, tiles, scales, dtype=torch.uint8, sdtype=BF, device="cpu"):
        return W4Weight(n, k, group, torch.zeros(tiles, dtype=dtype), torch.zeros(scales, dtype=sdtype, device=device))
    for n, k, group, tiles, scales in ((16, 64, 64, 512, 16), (17, 65, 32, 2048, 128), (1, 200, 128, 2048, 64)):
        w = make(n, k, group, tiles, scales)
        for bad in (dict(n=n + 16), dict(k=k + 64), dict(group=32 if group > 32 else 64), dict(n=0), dict(k=-1), dict(group=16),
                    dict(tiles=w.tiles[1:]), dict(scales=w.scales[1:]), dict(tiles=torch.zeros(2 * tiles, dtype=torch.uint8)[::2]),
                    dict(scales=torch.zeros(scales, dtype=BF, device="meta"))):
            with pytest.raises(ValueError):
                dataclasses.replace(w, **bad)
        for bad in (dict(tiles=w.tiles.to(torch.int32)), dict(scales=w.scales.float())):
            with pytest.raises(TypeError):
                dataclasses.replace(w, **bad)
