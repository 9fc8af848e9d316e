"""Block norms, host side: the C ABI's structures and argument checks (no
launch: the pointers are never read), and the refusal of CPU tensors."""

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
    a = N.LvsaBlockNorm()
    rows = N.LvsaRows(FAKE, 0, 64)
    a.x = a.y = a.h = a.n = rows
    a.next.kind, a.next.eps, a.post.kind = N.LVSA_BLOCK_NORM_LAYER, 1e-6, N.LVSA_BLOCK_NORM_NONE
    a.residual_scale, a.batch, a.seq, a.frames, a.width = 1.0, 1, 0, 1, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _fwd(a):
    return N.load().lvsa_block_norm_fwd(ctypes.byref(a), None)


def test_struct_layouts():
    probe = r'''
#include <stdio.h>
#include <stddef.h>
#include "lvsa_b200.h"
int main(void){
 printf("%zu %zu %zu %zu %zu %zu %zu %zu %zu\n", sizeof(LvsaRows), sizeof(LvsaVectors), sizeof(LvsaRowNorm),
        sizeof(LvsaBlockNorm), sizeof(LvsaBlockNormGrad), offsetof(LvsaBlockNorm, post),
        offsetof(LvsaBlockNorm, stats), offsetof(LvsaBlockNormGrad, dweight), offsetof(LvsaBlockNormGrad, workspace_bytes));
 return 0;}
'''
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
        with open(c, "w") as fh:
            fh.write(probe)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        got = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    size = ctypes.sizeof
    assert got == [size(N.LvsaRows), size(N.LvsaVectors), size(N.LvsaRowNorm), size(N.LvsaBlockNorm),
                   size(N.LvsaBlockNormGrad), N.LvsaBlockNorm.post.offset, N.LvsaBlockNorm.stats.offset,
                   N.LvsaBlockNormGrad.dweight.offset, N.LvsaBlockNormGrad.workspace_bytes.offset]


def test_forward_checks():
    assert _fwd(_args()) == N.LVSA_OK  # no rows: nothing to launch
    assert N.load().lvsa_block_norm_fwd(None, None) == N.LVSA_ERR_INVALID_ARG
    none = N.LvsaRows()
    assert _fwd(_args(x=none)) == N.LVSA_ERR_INVALID_ARG
    assert _fwd(_args(y=none, n=none)) == N.LVSA_ERR_INVALID_ARG
    assert _fwd(_args(h=none)) == N.LVSA_ERR_INVALID_ARG
    assert _fwd(_args(y=none, h=none)) == N.LVSA_OK
    for bad in (dict(batch=-1), dict(seq=-1), dict(frames=0), dict(width=0)):
        assert _fwd(_args(**bad)) == N.LVSA_ERR_INVALID_ARG, bad
    assert _fwd(_args(seq=7, frames=2)) == N.LVSA_ERR_GEOMETRY
    for bad in (dict(width=N.LVSA_BLOCK_NORM_MAX_WIDTH + 1), dict(stream_dtype=9), dict(branch_dtype=N.LVSA_DTYPE_E4M3),
                dict(batch=2, seq=2 ** 30), dict(stream_dtype=N.LVSA_DTYPE_BF16, branch_dtype=N.LVSA_DTYPE_F32),
                dict(gate=N.LvsaVectors(FAKE, 0, 0, N.LVSA_DTYPE_E4M3, 0))):
        assert _fwd(_args(**bad)) == N.LVSA_ERR_UNSUPPORTED, bad
    norm = N.LvsaRowNorm
    for bad in (dict(next=norm(0, 1e-6)), dict(next=norm(3, 1e-6)), dict(next=norm(1, -1.0)),
                dict(next=norm(1, float("nan"))), dict(next=norm(2, 0.0, 0, 0, None, FAKE)),
                dict(post=norm(0, 0.0, 0, 0, FAKE, None))):
        assert _fwd(_args(**bad)) == N.LVSA_ERR_INVALID_ARG, bad
    assert _fwd(_args(next=norm(1, 1e-6, 2, 0, FAKE, None))) == N.LVSA_ERR_UNSUPPORTED


def test_backward_checks():
    lib = N.load()

    def bwd(f, **kw):
        g = N.LvsaBlockNormGrad()
        g.f = f
        for k, v in kw.items():
            setattr(g, k, v)
        size = ctypes.c_int64(-1)
        st = lib.lvsa_block_norm_bwd(ctypes.byref(g), None)
        assert lib.lvsa_block_norm_workspace(ctypes.byref(g), ctypes.byref(size)) == st and size.value == 0
        return st
    full = dict(stats=FAKE, post_stats=FAKE)
    rows, none = N.LvsaRows(FAKE, 0, 64), N.LvsaRows()
    assert bwd(_args(**full), dn=rows) == N.LVSA_OK
    assert bwd(_args(), dn=rows) == N.LVSA_ERR_INVALID_ARG  # no statistics
    assert bwd(_args(stats=FAKE, post=N.LvsaRowNorm(2, 0.0)), dn=rows) == N.LVSA_ERR_INVALID_ARG
    assert bwd(_args(n=none), dn=rows) == N.LVSA_ERR_INVALID_ARG
    assert bwd(_args(y=none, **full), dh=rows) == N.LVSA_ERR_INVALID_ARG
    assert bwd(_args(**full), dweight=FAKE) == N.LVSA_ERR_INVALID_ARG  # no weight
    assert bwd(_args(**full), dpost_bias=FAKE) == N.LVSA_ERR_INVALID_ARG
    assert bwd(_args(**full), dgate=N.LvsaVectors(FAKE, 0, 0, 7, 0)) == N.LVSA_ERR_UNSUPPORTED
    assert lib.lvsa_block_norm_bwd(None, None) == N.LVSA_ERR_INVALID_ARG
    assert lib.lvsa_block_norm_workspace(None, None) == N.LVSA_ERR_INVALID_ARG


def test_cpu_tensors_are_refused():
    from longvideosparseattention_b200.block_norm import gate_residual, gate_residual_norm, norm_modulate
    x = torch.zeros(1, 2, 8)
    for call in (lambda: norm_modulate(x), lambda: gate_residual(x, x), lambda: gate_residual_norm(x, x)):
        with pytest.raises(RuntimeError):
            call()


def test_packed_arguments_have_the_structures_layout():
    """Fields packed as bytes fall where the C structures have them."""
    from longvideosparseattention_b200 import _launch as L
    for packer, struct in ((L.BLOCK_NORM, N.LvsaBlockNorm), (L.BLOCK_NORM_GRAD, N.LvsaBlockNormGrad),
                           (L.W4_LINEAR, N.LvsaW4Linear)):
        assert packer.size == ctypes.sizeof(struct)

        def leaves(s):
            for name, kind in s._fields_:
                v = getattr(s, name)
                yield from leaves(v) if isinstance(v, ctypes.Structure) else [0 if v is None else v]
        n = len(packer.unpack(bytes(packer.size)))
        values = list(range(1, n + 1))
        got = list(leaves(struct.from_buffer_copy(packer.pack(*values))))
        assert got == values[:len(got)] and n - len(got) in (0, 1)


def test_tangents_are_refused():
    """Where a level of forward-mode differentiation is entered, of dual tensors only."""
    from torch.autograd import forward_ad

    from longvideosparseattention_b200.block_norm import gate_residual_norm, norm_modulate
    from longvideosparseattention_b200._launch import refuse_tangents
    x, v = torch.zeros(1, 2, 8), torch.zeros(8)
    refuse_tangents("here", (x, None))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(v, torch.ones(8))
        for call in (lambda: refuse_tangents("here", (x, None, dual)), lambda: norm_modulate(x, scale=dual),
                     lambda: gate_residual_norm(x, x, dual)):
            with pytest.raises(NotImplementedError):
                call()
        refuse_tangents("here", (x, None, v))


def test_statistics_are_aligned():
    """A row's pair of statistics is one 8-byte access: a pointer between them is refused, with no rows too."""
    lib = N.load()
    rows = N.LvsaRows(FAKE, 0, 64)
    for where in ("stats", "post_stats"):
        kw = dict(stats=FAKE, post_stats=FAKE, post=N.LvsaRowNorm(2, 0.0))
        assert _fwd(_args(**kw)) == N.LVSA_OK
        kw[where] = FAKE + 4
        assert _fwd(_args(**kw)) == N.LVSA_ERR_ALIGNMENT
        g = N.LvsaBlockNormGrad()
        g.f, g.dn = _args(**kw), rows
        assert lib.lvsa_block_norm_bwd(ctypes.byref(g), None) == N.LVSA_ERR_ALIGNMENT
