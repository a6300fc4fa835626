"""The training-block operators' refusals and size queries, without a GPU: the Python checks raise ValueError before any
launch, the C ABI returns MZ_E_ARG with a message."""
import ctypes as C

import pytest
import torch

from muzero_amd import _lib, blocks

ONE = C.c_void_p(16)      # a non-null, 16-byte aligned address that is never dereferenced


def _fails(name, *args, match):
    with pytest.raises(_lib.MuZeroAmdError, match=match) as e:
        _lib.call(name, *args)
    assert name in str(e.value)


def test_tensors_have_to_live_on_the_gpu():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    for call in (lambda: blocks.layer_norm(x), lambda: blocks.gated_ff(x, w, w),
                 lambda: blocks.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for call in (lambda: blocks.layer_norm(None), lambda: blocks.dropout([1.0], 0.1, None)):
        with pytest.raises(ValueError, match="tensor required"):
            call()


def test_layer_norm_entry_points_refuse():
    fwd = lambda **k: [k.get(n, d) for n, d in dict(x=ONE, ldx=8, w=ONE, b=ONE, affine=0, eps=1e-5, rows=4, c=8, dt=1, y=ONE,  # noqa: E731
                                                    mean=ONE, rstd=ONE, s=None).items()]
    _fails("mz_layer_norm_fwd", *fwd(x=None), match="null")
    _fails("mz_layer_norm_fwd", *fwd(rstd=None), match="go together")
    _fails("mz_layer_norm_fwd", *fwd(rows=0), match="rows > 0")
    _fails("mz_layer_norm_fwd", *fwd(c=(1 << 24) + 1, ldx=1 << 25), match="rows > 0")
    _fails("mz_layer_norm_fwd", *fwd(ldx=7), match="overlap")
    _fails("mz_layer_norm_fwd", *fwd(dt=3), match="element type")
    _fails("mz_layer_norm_fwd", *fwd(affine=2), match="parameters")
    _fails("mz_layer_norm_fwd", *fwd(eps=-1.0), match="eps")
    _fails("mz_layer_norm_fwd", *fwd(eps=float("nan")), match="eps")
    bwd = lambda **k: [k.get(n, d) for n, d in dict(x=ONE, ldx=8, dy=ONE, lddy=8, w=ONE, affine=0, mean=ONE, rstd=ONE, rows=4,  # noqa: E731
                                                    c=8, dt=1, dx=ONE, dw=ONE, db=ONE, ws=ONE, nb=1 << 20, s=None).items()]
    _fails("mz_layer_norm_bwd", *bwd(mean=None), match="null")
    _fails("mz_layer_norm_bwd", *bwd(dx=None, dw=None, db=None), match="no gradient")
    _fails("mz_layer_norm_bwd", *bwd(lddy=4), match="overlap")
    _fails("mz_layer_norm_bwd", *bwd(nb=4 * 2 * 8 * 4 - 1), match="workspace")
    _fails("mz_layer_norm_bwd", *bwd(ws=None), match="workspace")
    lib = _lib.lib()
    assert lib.mz_layer_norm_workspace_bytes(4, 8) == 4 * 2 * 8 * 4
    assert lib.mz_layer_norm_workspace_bytes(1 << 20, 8) == 1024 * 2 * 8 * 4
    assert lib.mz_layer_norm_workspace_bytes(0, 8) == 0


def test_gated_ff_entry_points_refuse():
    fwd = lambda **k: [k.get(n, d) for n, d in dict(x=ONE, ldx=64, wg=ONE, wu=ONE, bg=None, bu=None, m=100, kk=64, f=32, dt=1,  # noqa: E731
                                                    act=0, h=ONE, ws=None, nb=0, s=None).items()]
    _fails("mz_gated_ff_fwd", *fwd(wu=None), match="null")
    _fails("mz_gated_ff_fwd", *fwd(act=4), match="activation")
    _fails("mz_gated_ff_fwd", *fwd(act=-1), match="activation")
    _fails("mz_gated_ff_fwd", *fwd(dt=7), match="element type")
    _fails("mz_gated_ff_fwd", *fwd(m=0), match="out of range")
    _fails("mz_gated_ff_fwd", *fwd(f=(1 << 20) + 1), match="out of range")
    _fails("mz_gated_ff_fwd", *fwd(ldx=63), match="stride")
    _fails("mz_gated_ff_fwd", *fwd(ldx=1 << 22), match="stride")
    bwd = lambda **k: [k.get(n, d) for n, d in dict(x=ONE, ldx=64, wg=ONE, wu=ONE, bg=None, bu=None, dh=ONE, m=100, kk=64, f=32,  # noqa: E731
                                                    dt=1, act=0, dx=ONE, dwg=ONE, dwu=ONE, dbg=None, dbu=None, ws=ONE,
                                                    nb=1 << 30, s=None).items()]
    _fails("mz_gated_ff_bwd", *bwd(dh=None), match="null")
    _fails("mz_gated_ff_bwd", *bwd(dwu=None), match="go together")
    _fails("mz_gated_ff_bwd", *bwd(dx=None, dwg=None, dwu=None), match="no gradient")
    need = _lib.lib().mz_gated_ff_workspace_bytes(100, 64, 32, 1, 1)
    assert need > 2 * 100 * 32 * 2
    _fails("mz_gated_ff_bwd", *bwd(nb=need - 1), match="workspace")
    _fails("mz_gated_ff_bwd", *bwd(ws=C.c_void_p(24)), match="16-byte aligned")
    lib = _lib.lib()
    assert lib.mz_gated_ff_workspace_bytes(100, 64, 32, 1, 0) == 0
    assert lib.mz_gated_ff_workspace_bytes(100, 63, 32, 1, 0) == 0
    assert lib.mz_gated_ff_workspace_bytes(1, 63, 32, 1, 0) == 0
    assert lib.mz_gated_ff_workspace_bytes(0, 64, 32, 1, 0) == -1


def test_dropout_entry_point_refuses():
    call = lambda **k: [k.get(n, d) for n, d in dict(x=ONE, r=None, y=ONE, n=8, p=0.1, rng=ONE, c=0, dt=0, s=None).items()]  # noqa: E731
    _fails("mz_dropout", *call(rng=None), match="null")
    _fails("mz_dropout", *call(n=0), match="elements")
    _fails("mz_dropout", *call(n=(1 << 35) + 1), match="elements")
    _fails("mz_dropout", *call(p=1.5), match=r"p in")
    _fails("mz_dropout", *call(p=float("nan")), match=r"p in")
    _fails("mz_dropout", *call(dt=3), match="element type")


def test_sizes_that_cannot_be_numbered_and_float_alignment():
    lib = _lib.lib()
    assert lib.mz_gated_ff_workspace_bytes(1 << 37, 1, 1, 1, 1) == -1
    assert lib.mz_gated_ff_workspace_bytes(1 << 36, 1 << 20, 1 << 20, 0, 1) > 0        # no overflow on the way
    _fails("mz_gated_ff_fwd", ONE, 64, ONE, ONE, None, None, 1 << 37, 64, 32, 1, 0, ONE, None, 0, None, match="out of range")
    _fails("mz_layer_norm_bwd", ONE, 8, ONE, 8, None, 0, ONE, ONE, 4, 8, 0, ONE, ONE, None, C.c_void_p(18), 1 << 20, None,
           match="aligned")


def test_layer_norm_workspace_is_what_the_launch_uses():
    """Partial rows of the workgroups that there can be, and a float a row where rows are wider than 16384 columns."""
    need = _lib.lib().mz_layer_norm_workspace_bytes
    assert need(1 << 20, 4096) == 1024 * 2 * 4096 * 4 and need(1 << 20, 4097) == 256 * 2 * 4097 * 4
    assert need(1 << 20, 16384) == 256 * 2 * 16384 * 4 and need(100, 16384) == 100 * 2 * 16384 * 4
    assert need(65536, 65536) == 32 * 2 * 65536 * 4 + 65536 * 4                 # not 537 MB
    assert need(1024, 1 << 24) == 1 * 2 * (1 << 24) * 4 + 1024 * 4              # not 137 GB
    assert need(3, 20000) == 3 * 2 * 20000 * 4 + 3 * 4


def test_strides_whose_bytes_pass_64_bits():
    """A stride of 2^62 elements is 2^64 or 2^63 bytes: out of range, not 0."""
    for ld in (1 << 62, (1 << 48) // 4 + 1):
        _fails("mz_layer_norm_fwd", ONE, ld, None, None, 0, 1e-5, 4, 8, 0, ONE, None, None, None, match="apart")
        _fails("mz_layer_norm_bwd", ONE, 8, ONE, ld, None, 0, ONE, ONE, 4, 8, 0, ONE, None, None, None, 0, None, match="apart")
    _fails("mz_layer_norm_fwd", ONE, 8, None, None, 0, 1e-5, 1 << 60, 8, 0, ONE, None, None, None, match="apart")
    for ldx in (1 << 62, 1 << 61, (1 << 63) - 1, (1 << 62) + 64, (1 << 61) + 64):
        for dt in (0, 1, 2):
            _fails("mz_gated_ff_fwd", ONE, ldx, ONE, ONE, None, None, 100, 64, 32, dt, 0, ONE, None, 0, None, match="stride")
            _fails("mz_gated_ff_bwd", ONE, ldx, ONE, ONE, None, None, ONE, 100, 64, 32, dt, 0, ONE, None, None, None, None, None, 1 << 30,
                   None, match="stride")
