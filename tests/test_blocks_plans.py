"""The gated feed-forward operator's kernels by the tile that they run in: every product in each of its tiles, alone and in a
launch with the other, cut and whole, against float64, with ragged edges on all sides.  Each case states what it is there for,
and the library is asked whether a call of its sizes still runs that."""
import ctypes as C

import pytest
import torch

from tests.test_blocks_gpu import TYPES, U, Canary, check_gated_ff, ff_inputs, ff_run, half, within

MZ = {"f32": 0, "bf16": 1, "f16": 2}


def plan_of(rows, k, f, t, want_dx=1, want_dw=1):
    """Tiles, cuts and launches of a call as a dict of sides and counts."""
    from muzero_amd import _lib
    p = (C.c_int32 * 8)()
    _lib.call("mz_gated_ff_plan", rows, k, f, MZ[t], want_dx, want_dw, p)
    return dict(zip(("forward", "gate", "dx", "dx_parts", "dw", "dw_parts", "together", "terms"), p))


# rows, K, F, type, what the plan has to be.  All of them odd: every edge of every tile is ragged.  cut: the sum is split
CASES = [
    (1483, 1695, 4519, "bf16", dict(forward=256, gate=256, dx=256, dx_parts="cut", dw=256, dw_parts=1, together=0)),
    (1483, 1695, 4519, "f16", dict(forward=256, gate=256, dx=256, dx_parts="cut", dw=256, dw_parts=1, together=0)),
    (16233, 999, 815, "bf16", dict(forward=256, gate=256, dx=256, dx_parts=1, dw=256, dw_parts="cut", together=0)),
    (16233, 999, 815, "f16", dict(forward=256, gate=256, dx=256, dx_parts=1, dw=256, dw_parts="cut", together=0)),
    (5343, 2633, 1291, "bf16", dict(forward=256, gate=256, dx=256, dx_parts=1, dw=128, dw_parts=1, together=0)),
    (2733, 2935, 2307, "f16", dict(forward=256, gate=256, dx=128, dx_parts=1, dw=256, dw_parts=1, together=0)),
    (10733, 1523, 773, "bf16", dict(forward=128, gate=128, dx=256, dx_parts=1, dw=128, dw_parts="cut", together=0)),
    (5089, 203, 931, "bf16", dict(forward=256, gate=64, dx=128, dx_parts="cut", dw=128, dw_parts="cut", together=1)),
    (16881, 209, 327, "f16", dict(forward=256, gate=256, dx=128, dx_parts=1, dw=128, dw_parts="cut", together=1)),
    (651, 107, 3791, "bf16", dict(forward=128, gate=128, dx=64, dx_parts="cut", dw=64, dw_parts=1, together=1)),
    (203, 107, 65, "f16", dict(forward=64, gate=64, dx=64, dx_parts=1, dw=64, dw_parts="cut", together=1, terms=1)),
    (103, 105, 61, "bf16", dict(forward=64, gate=64, dx=64, dx_parts="cut", dw=64, dw_parts="cut", together=1, terms=2)),
    (103, 1367, 71, "f16", dict(forward=64, gate=64, dx=64, dx_parts=1, dw=64, dw_parts=1, together=1, terms=2)),
    (957, 2015, 4037, "f32", dict(forward=128, gate=128, dx=128, dx_parts="cut", dw=128, dw_parts=1, together=0)),
    (7875, 951, 473, "f32", dict(forward=128, gate=128, dx=128, dx_parts=1, dw=128, dw_parts="cut", together=0)),
    (893, 255, 4655, "f32", dict(forward=128, gate=128, dx=128, dx_parts="cut", dw=128, dw_parts=1, together=1)),
    (14373, 105, 253, "f32", dict(forward=128, gate=128, dx=128, dx_parts=1, dw=128, dw_parts="cut", together=1)),
    (735, 271, 4797, "f32", dict(forward=128, gate=128, dx=64, dx_parts="cut", dw=64, dw_parts=1, together=0)),
    (9659, 295, 379, "f32", dict(forward=128, gate=128, dx=64, dx_parts=1, dw=64, dw_parts="cut", together=0)),
    (103, 109, 61, "f32", dict(forward=64, gate=64, dx=64, dx_parts="cut", dw=64, dw_parts="cut", together=1)),
]
IDS = ["%dx%dx%d-%s" % c[:4] for c in CASES]


@pytest.mark.parametrize("rows,k,f,t,want", CASES, ids=IDS)
def test_sizes_run_the_kernels_they_stand_for(rows, k, f, t, want):
    plan = plan_of(rows, k, f, t)
    assert {n: "cut" if v == "cut" and plan[n] > 1 else plan[n] for n, v in want.items()} == want, plan


def test_the_cases_cover_every_tile():
    """Each product in each tile there is (float32 has no 256), the gradients cut and whole, in a shared launch and their own."""
    for wide in (False, True):                  # 16-bit types; float32
        plans = [plan_of(*c[:4]) for c in CASES if (c[3] == "f32") == wide]
        sides = {64, 128} if wide else {64, 128, 256}
        for name in ("forward", "gate"):
            assert {p[name] for p in plans} == sides, (name, wide)
        for name in ("dx", "dw"):
            kinds = {(p[name], p[name + "_parts"] > 1, p["together"]) for p in plans}
            assert {k[0] for k in kinds if not k[2]} >= sides - {64}, (name, wide)
            assert {k[0] for k in kinds if k[2]} == {64, 128}, (name, wide)
            assert {k[1] for k in kinds if k[0] == max(sides)} == {True, False}, (name, wide)
    assert {plan_of(*c[:4])["terms"] for c in CASES if c[3] != "f32"} == {1, 2}
    assert plan_of(16, 64, 64, "bf16")["forward"] == 0 and plan_of(17, 64, 64, "bf16")["forward"] == 64


# gradients that are wanted without the other, at sizes where the cut for a launch of both is a bad one for that
ALONE = [
    (46983, 2393, 165, "bf16", "dw", dict(dw=256)), (18431, 255, 1023, "bf16", "dw", dict(dw=128)),
    (7517, 3247, 209, "f32", "dw", dict(dw=64)), (6179, 3937, 77, "f32", "dw", dict(dw=64)),
    (18431, 255, 1023, "f32", "dx", dict(dx=64)), (65535, 1023, 31, "f16", "dw", dict(dw=64)),
    (65535, 1023, 31, "f16", "dx", dict(dx=256)),
]


@pytest.mark.parametrize("rows,k,f,t,which,want", ALONE)
def test_a_gradient_alone_has_its_own_plan(rows, k, f, t, which, want):
    joint, alone = plan_of(rows, k, f, t), plan_of(rows, k, f, t, int(which == "dx"), int(which == "dw"))
    assert alone["together"] == 0 and {n: alone[n] for n in want} == want, alone
    assert (alone[which], alone[which + "_parts"]) != (joint[which], joint[which + "_parts"]) or joint["together"] == 0


def test_a_gradient_alone_has_the_joint_cut_where_little_is_gained():
    for rows, k, f, t in ((90, 64, 72, "bf16"), (90, 64, 72, "f32"), (300, 300, 300, "bf16"), (128, 256, 1024, "bf16")):
        joint, dx, dw = plan_of(rows, k, f, t), plan_of(rows, k, f, t, 1, 0), plan_of(rows, k, f, t, 0, 1)
        assert (dx["dx"], dx["dx_parts"], dw["dw"], dw["dw_parts"]) == (joint["dx"], joint["dx_parts"], joint["dw"], joint["dw_parts"])


def test_shared_launches_have_to_win_clearly_against_the_largest_tiles():
    for rows, k, f, together in ((46984, 2394, 166, 0), (4096, 1024, 4096, 0), (50344, 285, 473, 1), (500, 2000, 8000, 1)):
        assert plan_of(rows, k, f, "bf16")["together"] == together


def test_launches_stay_within_what_hip_can_count():
    """Threads of a launch are counted in 32 bits: 2^24 workgroups of 64 x 64 tiles are one too many, larger tiles take over; what
    no tile is large enough for is refused before anything is launched."""
    from muzero_amd import _lib
    assert plan_of(1 << 29, 1, 1, "bf16")["dx"] == 64 and plan_of((1 << 30) + 37, 1, 1, "bf16")["dx"] > 64
    assert plan_of(2 * 10 ** 9, 8, 8, "f32")["dx"] == 128 and plan_of(2 * 10 ** 9, 8, 8, "bf16")["dx"] > 64
    one = C.c_void_p(16)
    for rows, k, f, dt in ((1 << 33, 8, 8, 0), (1 << 34, 8, 8, 1), (1 << 36, 1 << 20, 1 << 20, 1)):
        for want in ((1, 0), (1, 1)):
            with pytest.raises(_lib.MuZeroAmdError, match="too many output tiles"):
                _lib.call("mz_gated_ff_plan", rows, k, f, dt, *want, (C.c_int32 * 8)())
        need = _lib.lib().mz_gated_ff_workspace_bytes(rows, k, f, dt, 1)
        with pytest.raises(_lib.MuZeroAmdError, match="mz_gated_ff_bwd.*too many output tiles"):
            _lib.call("mz_gated_ff_bwd", one, k, one, one, None, None, one, rows, k, f, dt, 0, one, None, None, None, None, one, need, None)
    with pytest.raises(_lib.MuZeroAmdError, match="mz_gated_ff_fwd.*too many output tiles"):
        _lib.call("mz_gated_ff_fwd", one, 8, one, one, None, None, 1 << 36, 8, 1 << 20, 1, 0, one, None, 0, None)


def test_plan_refuses():
    from muzero_amd import _lib
    p = (C.c_int32 * 8)()
    for args, match in (((0, 8, 8, 1, 1, 1, p), "out of range"), ((8, 8, (1 << 20) + 1, 1, 1, 1, p), "out of range"),
                        ((8, 8, 8, 3, 1, 1, p), "element type"), ((8, 8, 8, 1, 1, 1, None), "null")):
        with pytest.raises(_lib.MuZeroAmdError, match="mz_gated_ff_plan.*" + match):
            _lib.call("mz_gated_ff_plan", *args)
    assert plan_of(703, 263, 131, "bf16", 0, 1)["dx"] == 0 and plan_of(703, 263, 131, "bf16", 1, 0)["dw_parts"] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("rows,k,f,t,want", CASES, ids=IDS)
def test_every_tile_against_float64(rows, k, f, t, want, activation):
    x, wg, wu, bg, bu, dh = ff_inputs(rows + f, rows, k, f, TYPES[t], bias=activation != "relu")
    check_gated_ff(x, wg, wu, bg, bu, dh, activation, ff_run(x, wg, wu, bg, bu, dh, activation))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,f,t,want", CASES, ids=IDS)
def test_every_tile_writes_inside_its_buffers(rows, k, f, t, want):
    """Outputs and workspace between canaries, the workspace full of NaN; the same bits as the Python entry points."""
    from muzero_amd import _lib
    x, wg, wu, bg, bu, dh = ff_inputs(rows, rows, k, f, TYPES[t])
    p, s = (lambda v: v.data_ptr()), _lib.current_stream()
    want = ff_run(x, wg, wu, bg, bu, dh, "silu")
    out = [Canary(v.numel(), TYPES[t]) for v in want]
    need = _lib.lib().mz_gated_ff_workspace_bytes(rows, k, f, MZ[t], 1)
    ws = Canary((need + 3) // 4, torch.float32)
    _lib.call("mz_gated_ff_fwd", p(x), k, p(wg), p(wu), p(bg), p(bu), rows, k, f, MZ[t], 0, out[0].ptr(), None, 0, s)
    _lib.call("mz_gated_ff_bwd", p(x), k, p(wg), p(wu), p(bg), p(bu), p(dh), rows, k, f, MZ[t], 0, *(c.ptr() for c in out[1:]),
              ws.ptr(), need, s)
    assert (ws.all[:512] == 7.0).all() and (ws.all[-512:] == 7.0).all()
    for c, v in zip(out, want):
        c.check("gated_ff")
        assert torch.equal(c.inner, v.reshape(-1))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,f,t", [(16233, 999, 815, "bf16"), (7875, 951, 473, "f32"), (16881, 209, 327, "f16")])
def test_larger_tiles_strides_and_bad_values(rows, k, f, t):
    """Rows of x that lie apart, and a NaN in the last token and the last column of the ragged last tiles: everything else keeps
    its bits."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, wg, wu, bg, bu, dh = ff_inputs(rows, rows, k, f, TYPES[t])
    good = ff_run(x, wg, wu, bg, bu, dh, "silu")
    wide = torch.randn(rows, k + 45, generator=g, device="cuda").to(TYPES[t])
    wide[:, 13:13 + k] = x
    for a, b in zip(good, ff_run(wide[:, 13:13 + k], wg, wu, bg, bu, dh, "silu")):
        assert torch.equal(a, b)
    x[-1, -1] = float("nan")
    got = ff_run(x, wg, wu, bg, bu, dh, "silu")
    for i in (0, 1):
        assert torch.isnan(got[i][-1]).all() and torch.equal(got[i][:-1], good[i][:-1])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,f,t,which,want", ALONE)
def test_a_gradient_alone_against_float64(rows, k, f, t, which, want):
    """Frozen weights, or an input without a gradient; the workspace between canaries."""
    from muzero_amd import _lib, blocks
    x, wg, wu, bg, bu, dh = ff_inputs(rows, rows, k, f, TYPES[t])
    leaves = [v.detach().requires_grad_(v is x if which == "dx" else v is wg or v is wu) for v in (x, wg, wu, bg, bu)]
    h = blocks.gated_ff(*leaves)
    grads = torch.autograd.grad(h, [v for v in leaves if v.requires_grad], dh)
    parts = [grads[0], None, None] if which == "dx" else [None, grads[0], grads[1]]
    check_gated_ff(x, wg, wu, bg, bu, dh, "silu", [h.detach()] + parts + [None, None])
    p, s = (lambda v: v.data_ptr()), _lib.current_stream()
    need = _lib.lib().mz_gated_ff_workspace_bytes(rows, k, f, MZ[t], 1)
    ws, out = Canary((need + 3) // 4, torch.float32), [Canary(v.numel(), TYPES[t]) for v in grads]
    args = (out[0].ptr(), None, None) if which == "dx" else (None, out[0].ptr(), out[1].ptr())
    _lib.call("mz_gated_ff_bwd", p(x), k, p(wg), p(wu), p(bg), p(bu), p(dh), rows, k, f, MZ[t], 0, *args, None, None, ws.ptr(), need, s)
    assert (ws.all[:512] == 7.0).all() and (ws.all[-512:] == 7.0).all()
    for c, v in zip(out, grads):
        c.check(which)
        assert torch.equal(c.inner, v.reshape(-1))


@pytest.mark.gpu
def test_more_rows_than_the_smallest_tiles_can_number():
    """2^30 + 37 rows of one column: the last rows' results are a small call's, the gradient of the weight is theirs."""
    from muzero_amd import blocks
    t, rows, live = torch.bfloat16, (1 << 30) + 37, 37
    assert plan_of(rows, 1, 1, "bf16")["dx"] > 64
    g = torch.Generator(device="cuda").manual_seed(1)
    tail = torch.randn(live, 1, generator=g, device="cuda").to(t)
    x = torch.zeros(rows, 1, dtype=t, device="cuda")
    x[-live:] = tail
    wg, wu = (torch.randn(1, 1, generator=g, device="cuda").to(t).requires_grad_() for _ in range(2))
    dh = torch.zeros(rows, 1, dtype=t, device="cuda")
    dh[-live:] = 1.0
    x.requires_grad_()
    h = blocks.gated_ff(x, wg, wu)
    dx, dwg, dwu = torch.autograd.grad(h, (x, wg, wu), dh)
    assert torch.equal(h[-live:], blocks.gated_ff(tail, wg, wu)) and not h[:-live].any() and not dx[:-live].any()
    xd, gd, ud = tail.double(), wg.detach().double(), wu.detach().double()
    gate, up = xd @ gd.t(), xd @ ud.t()
    sig = torch.sigmoid(gate)
    dg, du = up * sig * (1 + gate * (1 - sig)), gate * sig
    # dg and du: off by their rounding, and by some 32 u of the activation's arithmetic (|gate| stays below 8)
    off = (half(t) + 32 * U) * 1.01
    e_dg, e_du = off * dg.abs() + 32 * U * up.abs() * (1 + gate.abs()), off * du.abs()
    within(dx[-live:], dg @ gd + du @ ud, e_dg @ gd.abs() + e_du @ ud.abs(), "dx")
    within(dwg, dg.t() @ xd, (e_dg + 40 * U * dg.abs()).t() @ xd.abs(), "dw_gate")
    within(dwu, du.t() @ xd, (e_du + 40 * U * du.abs()).t() @ xd.abs(), "dw_up")
