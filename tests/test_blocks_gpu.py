"""Layer norm, the gated feed-forward projection and dropout (muzero_amd.blocks) against their definitions in float64, at
the sizes, strides and values where they can go wrong.

Tolerances are bounds, not fits.  u = 2^-24 is float32's half step, `half(t)` the half step of the output type, relative
to the value.  A float32 sum of n terms added in any order is off by at most d u sum|terms| with d the number of
additions a term passes through (at most n)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half of the smallest step near zero (subnormal results are off by an absolute amount)."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, t=torch.float32, scale=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(t)


def within(got, ref, bound, what):
    bound = bound + half(got.dtype) * (ref.abs() + bound) + tiny(got.dtype)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got.double() - ref).abs() <= bound)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist(), got[bad][:3].tolist(), ref[bad][:3].tolist(),
                           bound[bad][:3].tolist())


# ------------------------------------------------------------------------------------------------------- layer norm
def check_layer_norm(x, w, b, dy, eps, got):
    """got: y, dx, dw, db (the last two or any may be None) for x [rows, C]."""
    y, dx, dw, db = got
    rows, c = x.shape
    xd, dyd = x.double(), dy.double()
    wd = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    mean = xd.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((xd - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (xd - mean) * rstd
    # A term of a row's sum passes through at most d additions: its thread's (16 columns, or C / 1024 of a wide row) and
    # a tree of 6 + 16.  mean: off by d u max|x|, so x - mean by (d + 2) u max|x|; the deviations enter the variance
    # squared and rstd takes half of their relative error: its own error is below (d + 4) u + the mean's share, squared.
    d = 24 + max(16, c / 1024)
    top = xd.abs().amax(1, keepdim=True)
    e_xh = (d + 2) * U * top * rstd + (2 * d + 8) * U * xh.abs()
    e_xh = e_xh + xh.abs() * ((d + 2) * U * top * rstd) ** 2
    within(y, xh * wd + bd, e_xh * wd.abs() + 3 * U * (xh * wd).abs() + 2 * U * bd.abs(), "y")
    if dx is not None:
        g = dyd * wd
        m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        e_m1 = (d + 2) * U * g.abs().mean(1, keepdim=True)
        e_m2 = (d + 4) * U * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
        inner = g.abs() + m1.abs() + (xh * m2).abs()
        e_dx = rstd * (e_m1 + xh.abs() * e_m2 + e_xh * m2.abs() + 6 * U * inner) + (2 * d + 10) * U * rstd * inner
        within(dx, rstd * (g - m1 - xh * m2), e_dx, "dx")
    # columns: a thread adds up to rows / 1 terms (few rows: few), the rest is a tree of at most 64
    dc = rows + 70
    if dw is not None:
        within(dw, (dyd * xh).sum(0), (dc * U * (dyd * xh).abs() + dyd.abs() * e_xh).sum(0), "dweight")
    if db is not None:
        within(db, dyd.sum(0), dc * U * dyd.abs().sum(0), "dbias")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,c", [(1, 1), (1, 256), (3, 7), (5, 8), (17, 100), (64, 129), (130, 256), (33, 511), (9, 600),
                                    (2000, 257), (7, 1001), (12, 2047), (4, 3000), (6, 4096), (3, 8190), (2, 16384), (3, 16385),
                                    (2, 40001), (1100, 24)])
def test_layer_norm_against_float64(rows, c, t):
    from muzero_amd import blocks
    t = TYPES[t]
    g = gen(rows * 31 + c)
    x = normal(g, rows, c, t=t, scale=2.0, mean=0.5).requires_grad_()
    for affine in {torch.float32, t}:
        w = normal(g, c, t=affine, scale=0.3, mean=1.0).requires_grad_()
        b = normal(g, c, t=affine, scale=0.3).requires_grad_()
        dy = normal(g, rows, c, t=t)
        y = blocks.layer_norm(x, w, b)
        assert y.dtype == t
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        assert dw.dtype == affine and db.dtype == affine
        check_layer_norm(x.detach(), w.detach(), b.detach(), dy, 1e-5, (y.detach(), dx, dw, db))
        with torch.no_grad():
            assert torch.equal(blocks.layer_norm(x, w, b), y)


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_layer_norm_parts_strides_and_leading_shapes(t):
    """Without weight or bias, with one gradient wanted at a time, on rows that lie apart, on transposed and expanded
    tensors, with a gradient of stride 0."""
    from muzero_amd import blocks
    t = TYPES[t]
    g = gen(3)
    wide = normal(g, 6, 5, 300, t=t)
    w, b = normal(g, 100, t=t, mean=1.0), normal(g, 100, t=t)
    for x in (wide[:, :, 100:200], wide[:, :, 1:101], wide.transpose(0, 1)[:, :, :100], wide[:, 0, :100],
              wide[0, 0, :100], wide[0, 0, :100].expand(4, 100), wide.permute(2, 0, 1)[:100].permute(1, 2, 0)):
        flat = x.reshape(-1, 100).contiguous()
        dy = normal(g, *x.shape, t=t)
        for ww, bb in ((w, b), (None, b), (w, None), (None, None)):
            leaf = x.detach().requires_grad_()
            ww, bb = (None if p is None else p.detach().requires_grad_() for p in (ww, bb))
            y = blocks.layer_norm(leaf, ww, bb, eps=1e-3)
            wrt = [p for p in (leaf, ww, bb) if p is not None]
            grads = dict(zip(map(id, wrt), torch.autograd.grad(y, wrt, dy)))
            parts = [None if p is None else grads[id(p)] for p in (leaf, ww, bb)]
            check_layer_norm(flat, ww, bb, dy.reshape(-1, 100), 1e-3,
                             (y.detach().reshape(-1, 100), parts[0].reshape(-1, 100), parts[1], parts[2]))
            for p in wrt:               # each alone: the same bits
                alone = torch.autograd.grad(blocks.layer_norm(leaf, ww, bb, eps=1e-3), p, dy)[0]
                assert torch.equal(alone, grads[id(p)])
    leaf = flat.requires_grad_()
    y = blocks.layer_norm(leaf, w, b)
    ones = torch.autograd.grad(y, leaf, torch.ones(1, 1, dtype=t, device="cuda").expand_as(y))[0]
    assert torch.equal(ones, torch.autograd.grad(blocks.layer_norm(leaf, w, b), leaf, torch.ones_like(y))[0])


def test_layer_norm_large_offset_constant_rows_and_bad_values():
    """A common offset of 1e4 standard deviations costs the digits float32 x itself has lost, not more; constant rows give
    the bias; a NaN or an infinity stays in its row."""
    from muzero_amd import blocks
    g = gen(4)
    x = normal(g, 40, 777, mean=1e4)
    w, b = normal(g, 777, mean=1.0), normal(g, 777)
    dy = normal(g, 40, 777)
    leaf = x.clone().requires_grad_()
    y = blocks.layer_norm(leaf, w, b)
    check_layer_norm(x, w, b, dy, 1e-5, (y.detach(), torch.autograd.grad(y, leaf, dy)[0], None, None))
    flat = torch.full((3, 64), 2.5, device="cuda")
    assert torch.equal(blocks.layer_norm(flat, None, b[:64].contiguous()), b[:64].expand(3, 64))
    x = normal(g, 40, 777)
    good = blocks.layer_norm(x, w, b)
    x[7, 5], x[23, 700], x[31] = float("nan"), float("inf"), float("-inf")
    y = blocks.layer_norm(x, w, b)
    bad = torch.tensor([r in (7, 23, 31) for r in range(40)], device="cuda")
    assert torch.isnan(y[7]).all() and torch.equal(y[~bad], good[~bad])


def test_layer_norm_no_rows():
    from muzero_amd import blocks
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = blocks.layer_norm(x, w, None)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 16, device="cuda"))
    assert y.shape == (0, 16) and dx.shape == (0, 16) and torch.equal(dw, torch.zeros(16, device="cuda"))


# ------------------------------------------------------------------------------------------- gated feed-forward
ACT = {
    "silu": (lambda v: v * torch.sigmoid(v), lambda v: torch.sigmoid(v) * (1 + v * (1 - torch.sigmoid(v))), 0.5),
    "gelu": (lambda v: 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5)),
             lambda v: 0.5 * (1 + torch.erf(v * 0.5 ** 0.5)) + v * torch.exp(-0.5 * v * v) / (2 * np.pi) ** 0.5, 0.8),
    "relu": (lambda v: v.clamp(min=0), lambda v: (v > 0).double(), 0.0),
    "sigmoid": (torch.sigmoid, lambda v: torch.sigmoid(v) * (1 - torch.sigmoid(v)), 0.1),
}


def check_gated_ff(x, wg, wu, bg, bu, dh, activation, got):
    """got: h, dx, dwg, dwu, dbg, dbu (None: not checked), x [rows, K]."""
    t = x.dtype
    act, slope, curve = ACT[activation]          # curve bounds |act''|; |act'| <= 1.13
    xd, gd, ud = x.double(), wg.double(), wu.double()
    k, f, m = x.shape[1], wg.shape[0], x.shape[0]
    gate, up = xd @ gd.t(), xd @ ud.t()
    e_g, e_u = (k + 1) * U * (xd.abs() @ gd.abs().t()), (k + 1) * U * (xd.abs() @ ud.abs().t())
    if bg is not None:
        gate, e_g = gate + bg.double(), e_g + U * (gate.abs() + bg.double().abs())
    if bu is not None:
        up, e_u = up + bu.double(), e_u + U * (up.abs() + bu.double().abs())
    # the activation's own arithmetic: 16-bit types use the hardware's exponential, off by up to |gate| 2^-23 relative
    # where it matters, plus the reciprocal's and a handful of roundings; float32 the library's
    rel = 12 * U if t == torch.float32 else 16 * U + 2 * U * gate.abs()
    a, s = act(gate), slope(gate)
    e_a = 1.13 * e_g + rel * (a.abs() + (0.5 * gate.abs() if activation == "gelu" else 0))
    e_s = curve * e_g + rel * (1.13 + gate.abs())
    if activation == "relu":                     # the step at zero: either side of it is right within e_g
        e_s = e_s + (gate.abs() <= e_g).double()
    h, dx, dwg, dwu, dbg, dbu = got
    within(h, a * up, e_a * up.abs() + a.abs() * e_u + e_a * e_u + 2 * U * (a * up).abs(), "h")
    if dh is None:
        return
    dhd = dh.double()
    dg, du = dhd * up * s, dhd * a
    e_dg = dhd.abs() * (up.abs() * e_s + e_u * s.abs() + e_u * e_s) + 3 * U * dg.abs()
    e_du = dhd.abs() * e_a + 2 * U * du.abs()
    r_dg, r_du = e_dg, e_du                      # rounded to the operands' type for the products, not for the biases
    if t != torch.float32:
        step = half(t) if m * f > 8192 else half(t) ** 2         # few: in two parts, the second rounded
        r_dg = e_dg + step * (dg.abs() + e_dg) + tiny(t)
        r_du = e_du + step * (du.abs() + e_du) + tiny(t)
    if dx is not None:
        size = dg.abs() @ gd.abs() + du.abs() @ ud.abs()
        within(dx, dg @ gd + du @ ud, r_dg @ gd.abs() + r_du @ ud.abs() + (2 * f + 40) * U * size * 1.01, "dx")
    for out, v, r, name in ((dwg, dg, r_dg, "dw_gate"), (dwu, du, r_du, "dw_up")):
        if out is not None:
            within(out, v.t() @ xd, r.t() @ xd.abs() + (m + 40) * U * (v.abs().t() @ xd.abs()) * 1.01, name)
    for out, v, e, name in ((dbg, dg, e_dg, "db_gate"), (dbu, du, e_du, "db_up")):
        if out is not None:
            within(out, v.sum(0), (e + (m + 1) * U * v.abs()).sum(0), name)


def ff_inputs(seed, rows, k, f, t, bias=True):
    g = gen(seed)
    x, dh = normal(g, rows, k, t=t), normal(g, rows, f, t=t, scale=0.3)
    wg, wu = normal(g, f, k, t=t, scale=k ** -0.5), normal(g, f, k, t=t, scale=k ** -0.5)
    bg, bu = (normal(g, f, t=t, scale=0.3), normal(g, f, t=t, scale=0.3)) if bias else (None, None)
    return x, wg, wu, bg, bu, dh


def ff_run(x, wg, wu, bg, bu, dh, activation):
    from muzero_amd import blocks
    leaves = [None if p is None else p.detach().requires_grad_() for p in (x, wg, wu, bg, bu)]
    h = blocks.gated_ff(*leaves, activation=activation)
    grads = iter(torch.autograd.grad(h, [p for p in leaves if p is not None], dh))
    return [h.detach()] + [None if p is None else next(grads) for p in leaves]


# rows: one, the streaming kernel's three sizes and its end, tile edges, a cut sum; K: below one 16-byte unit, odd, no
# whole unit, whole steps and not; F likewise
FF_SHAPES = [(1, 1, 1), (1, 256, 1024), (2, 7, 5), (16, 64, 33), (17, 96, 40), (33, 130, 48), (64, 257, 65), (65, 64, 64),
             (66, 33, 20), (128, 256, 128), (129, 264, 130), (300, 72, 1000), (1000, 257, 1001), (513, 520, 264), (4100, 64, 24),
             (777, 8, 8), (2500, 512, 136), (300, 1, 200), (300, 2, 101), (200, 3, 70), (129, 5, 9), (70, 6, 16), (66, 4, 7),
             (1, 4096, 300), (3, 300, 2500), (40, 1001, 200), (8, 136, 1024)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k,f", FF_SHAPES)
def test_gated_ff_against_float64(rows, k, f, t):
    x, wg, wu, bg, bu, dh = ff_inputs(rows + k + f, rows, k, f, TYPES[t], bias=(rows + f) % 3 != 0)
    activation = list(ACT)[(rows + k) % 4]
    check_gated_ff(x, wg, wu, bg, bu, dh, activation, ff_run(x, wg, wu, bg, bu, dh, activation))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k,f", [(4200, 320, 2200), (2304, 1100, 1100)])
def test_gated_ff_largest_tiles_against_float64(rows, k, f, t):
    """Sizes at which every product takes its largest tiles, ragged in all three."""
    x, wg, wu, bg, bu, dh = ff_inputs(rows, rows, k, f, TYPES[t])
    check_gated_ff(x, wg, wu, bg, bu, dh, "silu", ff_run(x, wg, wu, bg, bu, dh, "silu"))


@pytest.mark.parametrize("activation", ACT)
@pytest.mark.parametrize("t", TYPES)
def test_gated_ff_activations_far_from_zero(activation, t):
    """Gates of +-200 (an exponential beyond float32 on one side): finite results, the definition's."""
    t = TYPES[t]
    x, wg, wu, bg, bu, dh = ff_inputs(5, 70, 64, 72, t)
    wg = (wg.float() * 60).to(t)
    got = ff_run(x, wg, wu, bg, bu, dh, activation)
    assert all(torch.isfinite(v.float()).all() for v in got)
    check_gated_ff(x, wg, wu, bg, bu, dh, activation, got)


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_gated_ff_strides_parts_and_one_bias(t):
    """Rows that lie apart (aligned: read in place; not: copied), transposed weights, one bias only, one gradient at a
    time (the same bits), a gradient of stride 0."""
    from muzero_amd import blocks
    t = TYPES[t]
    x, wg, wu, bg, bu, dh = ff_inputs(6, 90, 64, 72, t)
    wide = normal(gen(7), 90, 200, t=t)
    for xs in (wide[:, 64:128], wide[:, 3:67], wide.t()[:64].t(), wide[:1, :64].expand(90, 64), wide[::2, 8:72]):
        n = xs.shape[0]
        check_gated_ff(xs.contiguous(), wg, wu, bg, bu, dh[:n], "silu", ff_run(xs, wg, wu, bg, bu, dh[:n], "silu"))
    wt = wg.t().contiguous().t()
    both = ff_run(x, wt, wu, bg, None, dh, "gelu")
    check_gated_ff(x, wg, wu, bg, None, dh, "gelu", both)
    check_gated_ff(x, wg, wu, None, bu, dh, "gelu", ff_run(x, wg, wu, None, bu, dh, "gelu"))
    full = ff_run(x, wg, wu, bg, bu, dh, "silu")
    for i in range(5):
        leaves = [p.detach().requires_grad_(i == j) for j, p in enumerate((x, wg, wu, bg, bu))]
        alone = torch.autograd.grad(blocks.gated_ff(*leaves), leaves[i], dh)[0]
        assert torch.equal(alone, full[1 + i]), i
    leaf = x.detach().requires_grad_()
    one = torch.autograd.grad(blocks.gated_ff(leaf, wg, wu).sum(), leaf)[0]
    assert torch.equal(one, torch.autograd.grad(blocks.gated_ff(leaf, wg, wu), leaf, torch.ones_like(dh))[0])


def test_gated_ff_leading_shapes_no_rows_and_autocast():
    from muzero_amd import blocks
    x, wg, wu, bg, bu, dh = ff_inputs(8, 24, 32, 40, torch.bfloat16)
    h = blocks.gated_ff(x, wg, wu, bg, bu)
    assert torch.equal(blocks.gated_ff(x.view(2, 3, 4, 32), wg, wu, bg, bu), h.view(2, 3, 4, 40))
    assert torch.equal(blocks.gated_ff(x[0], wg, wu, bg, bu), blocks.gated_ff(x[:1], wg, wu, bg, bu)[0])
    with torch.autocast("cuda", dtype=torch.bfloat16):      # float32 parameters, as the learner's modules hold them
        w32 = wg.float().requires_grad_()
        ha = blocks.gated_ff(x, w32, wu.float(), bg.float(), bu.float())
    assert torch.equal(ha, h)
    d32 = torch.autograd.grad(ha, w32, dh)[0]
    assert d32.dtype == torch.float32
    empty = torch.empty(0, 32, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    leaf = wg.clone().requires_grad_()
    h0 = blocks.gated_ff(empty, leaf, wu)
    dx, dw = torch.autograd.grad(h0, (empty, leaf), torch.empty_like(h0))
    assert h0.shape == (0, 40) and dx.shape == (0, 32) and not dw.any()


def test_gated_ff_bad_values_stay_in_their_rows_and_features():
    """A NaN in one token, an infinity in one weight row: everything else keeps its bits (a ragged tile must not let them
    reach across its edge)."""
    from muzero_amd import blocks
    for t in (torch.bfloat16, torch.float32):
        x, wg, wu, bg, bu, dh = ff_inputs(9, 100, 72, 70, t)
        good = ff_run(x, wg, wu, bg, bu, dh, "silu")
        xb = x.clone()
        xb[99, 71] = float("nan")
        got = ff_run(xb, wg, wu, bg, bu, dh, "silu")
        assert torch.isnan(got[0][99]).all() and torch.equal(got[0][:99], good[0][:99])
        assert torch.isnan(got[1][99]).all() and torch.equal(got[1][:99], good[1][:99])
        wb = wg.clone()
        wb[69, 0] = float("inf")
        h = blocks.gated_ff(x, wb, wu, bg, bu)
        assert torch.equal(h[:, :69], good[0][:, :69])


# ---------------------------------------------------------------------------------------------------------- dropout
def keep_mask(seed, offset, call, n, p):
    """Philox4x32-10 in Python integers over numpy arrays."""
    m = 0xffffffff
    block = np.arange((n + 7) // 8, dtype=np.uint64)
    c = [block, np.full_like(block, call), np.full_like(block, offset & m), np.full_like(block, (offset >> 32) & m)]
    k0, k1 = seed & m, (seed >> 32) & m
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        s = np.uint64(32)
        c = [(p1 >> s) ^ c[1] ^ np.uint64(k0), p1 & np.uint64(m), (p0 >> s) ^ c[3] ^ np.uint64(k1), p0 & np.uint64(m)]
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    words = np.stack(c, 1)
    bits = np.stack([words & np.uint64(0xffff), words >> np.uint64(16)], 2).reshape(-1)[:n]
    return torch.from_numpy((bits >= np.uint64(round(p * 65536))).copy()).cuda()


def check_dropout(x, residual, keep, p, y):
    scale = 65536 / (65536 - round(p * 65536)) if round(p * 65536) < 65536 else 0.0
    kept = torch.where(keep.view(x.shape), x.double() * scale, 0.0)
    ref = kept if residual is None else kept + residual.double()
    within(y, ref, 2 * U * kept.abs() + U * ref.abs(), "dropout")


def test_dropout_generator_matches_a_published_vector():
    """The test's own generator at a known answer of Philox4x32-10: counter 0, key 0 -> 6627e8d5 e169c58d bc57ac4c 9b00dbd8
    (Random123's kat_vectors)."""
    want = [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    halves = [h for w in want for h in (w & 0xffff, w >> 16)]
    for i, h in enumerate(halves):              # element i is kept at p = h / 65536 and dropped one step later
        assert bool(keep_mask(0, 0, 0, 8, h / 65536)[i]) and not bool(keep_mask(0, 0, 0, 8, (h + 1) / 65536)[i])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5, 11), (128, 256), (1000, 257), (70001,)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_dropout_against_the_definition(shape, t, with_residual):
    from muzero_amd import blocks
    t = TYPES[t]
    g = gen(len(shape) + shape[0])
    x = normal(g, *shape, t=t).requires_grad_()
    residual = normal(g, *shape, t=t).requires_grad_() if with_residual else None
    dy = normal(g, *shape, t=t)
    seed, offset, call = 0x123456789abcdef, (5 << 32) + 77, 3000000001
    rng = torch.tensor([seed, offset], dtype=torch.int64, device="cuda")
    for p in (0.0, 0.1, 0.5, 0.999, 1.0):
        keep = keep_mask(seed, offset, call, x.numel(), p)
        y = blocks.dropout(x, p, rng, call, residual)
        check_dropout(x.detach(), None if residual is None else residual.detach(), keep, p, y.detach())
        wrt = [x] if residual is None else [x, residual]
        grads = torch.autograd.grad(y, wrt, dy)
        check_dropout(dy, None, keep, p, grads[0])
        assert residual is None or torch.equal(grads[1], dy)
    y = blocks.dropout(x.detach(), 0.3, rng, call)
    assert not torch.equal(y, blocks.dropout(x.detach(), 0.3, rng, call + 1)) or x.numel() < 20
    assert not torch.equal(y, blocks.dropout(x.detach(), 0.3, rng + 1, call)) or x.numel() < 20


def test_dropout_rate_and_independence():
    """2^22 elements: the share kept within five standard deviations of 1 - p, as is the share kept in both of two calls
    and in both of two neighbours."""
    from muzero_amd import blocks
    n, p = 1 << 22, 0.3
    x = torch.ones(n, device="cuda")
    rng = torch.tensor([99, 0], dtype=torch.int64, device="cuda")
    a, b = blocks.dropout(x, p, rng, 0) != 0, blocks.dropout(x, p, rng, 1) != 0
    for share, q in ((a, 0.7), (a & b, 0.49), (a[1:] & a[:-1], 0.49)):
        # neighbours overlap in pairs, which at most triples the variance
        assert abs(share.double().mean().item() - q) < 5 * (3 * q * (1 - q) / n) ** 0.5 + 2.0 ** -16


def test_dropout_bad_values_strides_and_changed_state():
    from muzero_amd import blocks
    rng = torch.tensor([4, 4], dtype=torch.int64, device="cuda")
    keep = keep_mask(4, 4, 0, 600, 0.5).view(20, 30)
    for bad in (float("nan"), float("inf"), float("-inf")):
        x = torch.full((20, 30), bad, device="cuda")
        y = blocks.dropout(x, 0.5, rng, residual=torch.ones_like(x))
        assert (y[~keep] == 1.0).all() and not torch.isfinite(y[keep]).any()
    x = normal(gen(1), 30, 20)
    assert torch.equal(blocks.dropout(x.t(), 0.5, rng), blocks.dropout(x.t().contiguous(), 0.5, rng))
    flat = normal(gen(2), 601)
    assert torch.equal(blocks.dropout(flat[1:], 0.5, rng), blocks.dropout(flat[1:].clone(), 0.5, rng))
    leaf = x.clone().requires_grad_()
    y = blocks.dropout(leaf, 0.5, rng)
    rng += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert blocks.dropout(torch.empty(0, 4, device="cuda"), 0.5, rng).shape == (0, 4)


# --------------------------------------------------------------------------------------------------------- refusals
def test_refusals():
    from muzero_amd import blocks
    x, w, v = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda"), torch.zeros(8, device="cuda")
    rng = torch.zeros(2, dtype=torch.int64, device="cuda")
    cases = [
        (lambda: blocks.layer_norm(x.double()), "dtype"), (lambda: blocks.layer_norm(x.long()), "dtype"),
        (lambda: blocks.layer_norm(x[:, :0]), "at least 1"), (lambda: blocks.layer_norm(x.sum()), "at least 1"),
        (lambda: blocks.layer_norm(x, v[:7]), "shape"), (lambda: blocks.layer_norm(x, v.half()), "dtype"),
        (lambda: blocks.layer_norm(x, v, v.cpu()), "on cpu"), (lambda: blocks.layer_norm(x, eps=-1.0), "eps"),
        (lambda: blocks.layer_norm(x.bfloat16(), v, v.bfloat16()), "dtype"), (lambda: blocks.layer_norm(x, eps=float("nan")), "eps"),
        (lambda: blocks.gated_ff(x, w, w, activation="tanh"), "activation"), (lambda: blocks.gated_ff(x, w, w[:5]), "shape"),
        (lambda: blocks.gated_ff(x, w.half(), w.half()), "dtype"), (lambda: blocks.gated_ff(x, w, w, v), "shape"),
        (lambda: blocks.gated_ff(x[:, :7], w, w), "shape"), (lambda: blocks.gated_ff(x, v, v), "F, K"),
        (lambda: blocks.gated_ff(x, w[:0], w[:0]), "at least 1"), (lambda: blocks.gated_ff(x, w, None), "tensor required"),
        (lambda: blocks.gated_ff(x, w.cpu(), w), "on cpu"), (lambda: blocks.dropout(x, 1.5, rng), "p 1.5"),
        (lambda: blocks.dropout(x, float("nan"), rng), "p nan"), (lambda: blocks.dropout(x, 0.5, rng.int()), "dtype"),
        (lambda: blocks.dropout(x, 0.5, rng.cpu()), "on cpu"), (lambda: blocks.dropout(x, 0.5, rng, call=-1), "call"),
        (lambda: blocks.dropout(x, 0.5, rng, call=1 << 32), "call"), (lambda: blocks.dropout(x, 0.5, rng, residual=v), "shape"),
        (lambda: blocks.dropout(x, 0.5, rng, residual=x.half()), "dtype"), (lambda: blocks.dropout(x, 0.5, None), "rng"),
        (lambda: blocks.dropout(x, 0.5, torch.zeros(4, dtype=torch.int64, device="cuda")[::2]), "contiguous"),
    ]
    for call, match in cases:
        with pytest.raises(ValueError, match=match):
            call()
    leaf = x.clone().requires_grad_()
    first = torch.autograd.grad(blocks.layer_norm(leaf).sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiat|once_differentiable|grad"):
        torch.autograd.grad(first.sum(), leaf)


# ----------------------------------------------------------------------------- bounds of what is written; large offsets
class Canary:
    """A buffer of n elements between margins of a known value."""

    def __init__(self, n, t, margin=512):
        self.all = torch.full((n + 2 * margin,), 7.0, dtype=t, device="cuda")
        self.inner, self.margin = self.all[margin:margin + n], margin
        self.inner.fill_(float("nan"))

    def ptr(self):
        return self.inner.data_ptr()

    def check(self, what):
        assert (self.all[:self.margin] == 7.0).all() and (self.all[-self.margin:] == 7.0).all(), what
        assert not torch.isnan(self.inner.float()).any(), what


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k,f", [(5, 40, 33), (100, 64, 33), (130, 37, 70), (700, 264, 130)])
def test_outputs_and_workspaces_stay_inside_their_buffers(rows, k, f, t):
    """Through the C ABI, outputs and workspace between canaries, the workspace full of NaN: everything asked for is
    written, nothing outside, and the results are those of the Python entry points."""
    from muzero_amd import _lib, blocks
    t = TYPES[t]
    dt = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[t]          # MZ_F32, MZ_BF16, MZ_F16
    x, wg, wu, bg, bu, dh = ff_inputs(rows, rows, k, f, t)
    p, s = (lambda v: v.data_ptr()), _lib.current_stream()
    want = ff_run(x, wg, wu, bg, bu, dh, "silu")
    out = [Canary(v.numel(), t) for v in want]
    for back in (0, 1):
        need = _lib.lib().mz_gated_ff_workspace_bytes(rows, k, f, dt, back)
        ws = Canary((need + 3) // 4, torch.float32)
        if back:
            _lib.call("mz_gated_ff_bwd", p(x), k, p(wg), p(wu), p(bg), p(bu), p(dh), rows, k, f, dt, 0,
                      *(c.ptr() for c in out[1:]), ws.ptr(), need, s)
        else:
            _lib.call("mz_gated_ff_fwd", p(x), k, p(wg), p(wu), p(bg), p(bu), rows, k, f, dt, 0, out[0].ptr(), ws.ptr(), need, s)
        assert (ws.all[:512] == 7.0).all() and (ws.all[-512:] == 7.0).all()
    for c, v in zip(out, want):
        c.check("gated_ff")
        assert torch.equal(c.inner, v.reshape(-1))
    # layer norm and dropout on the same tensors
    y, stats = Canary(rows * k, t), Canary(2 * rows, torch.float32)
    dx, dw, db = Canary(rows * k, t), Canary(k, torch.float32), Canary(k, torch.float32)
    w = torch.rand(k, device="cuda")
    need = _lib.lib().mz_layer_norm_workspace_bytes(rows, k)
    ws = Canary(need // 4, torch.float32)
    _lib.call("mz_layer_norm_fwd", p(x), k, p(w), p(w), 0, 1e-5, rows, k, dt, y.ptr(), stats.ptr(), stats.ptr() + 4 * rows, s)
    _lib.call("mz_layer_norm_bwd", p(x), k, p(x), k, p(w), 0, stats.ptr(), stats.ptr() + 4 * rows, rows, k, dt, dx.ptr(),
              dw.ptr(), db.ptr(), ws.ptr(), need, s)
    assert (ws.all[:512] == 7.0).all() and (ws.all[-512:] == 7.0).all()
    rng = torch.zeros(2, dtype=torch.int64, device="cuda")
    z = Canary(rows * k, t)
    _lib.call("mz_dropout", p(x), p(x), z.ptr(), rows * k, 0.2, p(rng), 0, dt, s)
    for c in (y, stats, dx, dw, db, z):
        c.check("layer norm, dropout")
    assert torch.equal(z.inner.view(rows, k), blocks.dropout(x, 0.2, rng, residual=x))


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows equal those of a small call (layer norm, gated_ff) and the definition
    (dropout); the gradients of parameters whose other rows are zero equal the small call's."""
    from muzero_amd import blocks
    t = torch.bfloat16
    rows, c, live = (1 << 21) + 37, 1032, 37                     # 2.16e9 elements
    g = gen(11)
    tail = normal(g, live, c, t=t)
    x = torch.zeros(rows, c, dtype=t, device="cuda")
    x[-live:] = tail
    w = normal(g, c, mean=1.0)
    y = blocks.layer_norm(x, w)
    assert torch.equal(y[-live:], blocks.layer_norm(tail, w)) and not y[:live].any()
    leaf = x.requires_grad_()
    dx, = torch.autograd.grad(blocks.layer_norm(leaf, w), leaf, x.detach())
    small = tail.clone().requires_grad_()
    assert torch.equal(dx[-live:], torch.autograd.grad(blocks.layer_norm(small, w), small, tail)[0])
    del y, dx, leaf
    x = x.detach()
    rng = torch.tensor([1, 2], dtype=torch.int64, device="cuda")
    x.fill_(1.0)
    y = blocks.dropout(x, 0.5, rng).view(-1)
    n = y.numel()
    first = (n - 4096) // 8 * 8
    keep = torch.cat([keep_tail(1, 2, first, n, 0.5)])
    assert torch.equal(y[first:] != 0, keep)
    del y, x
    xs = torch.zeros(rows, 16, dtype=t, device="cuda")
    xs[-live:] = tail[:, :16]
    wg, wu = normal(g, c, 16, t=t), normal(g, c, 16, t=t)
    wg.requires_grad_(), wu.requires_grad_()
    dh = torch.ones(1, 1, dtype=t, device="cuda").expand(rows, c)
    leaf = xs.requires_grad_()
    h = blocks.gated_ff(leaf, wg, wu)
    small = tail[:, :16].contiguous().repeat(3, 1).requires_grad_()    # more than the streaming kernel's rows
    hs = blocks.gated_ff(small, wg, wu)
    assert torch.equal(h[-live:], hs[:live]) and not h[:live].any()
    dx, dwg = torch.autograd.grad(h, (leaf, wg), dh)
    ds, dwgs = torch.autograd.grad(hs, (small, wg), torch.ones_like(hs))
    # the small call may cut its sum over the features into parts: the same terms, rounded differently
    assert (dx[-live:].double() - ds[:live].double()).abs().max() <= 2 * half(t) * ds.abs().max().double()
    assert (dwg.double() * 3 - dwgs.double()).abs().max() <= 4 * half(t) * dwgs.abs().max().double()


def keep_tail(seed, offset, first, n, p):
    """keep_mask of elements first .. n (first a multiple of 8)."""
    m = 0xffffffff
    block = np.arange(first // 8, (n + 7) // 8, dtype=np.uint64)
    s = np.uint64(32)
    c = [block, np.zeros_like(block), np.full_like(block, offset & m), np.full_like(block, offset >> 32)]
    k0, k1 = seed & m, seed >> 32
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> s) ^ c[1] ^ np.uint64(k0), p1 & np.uint64(m), (p0 >> s) ^ c[3] ^ np.uint64(k1), p0 & np.uint64(m)]
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    words = np.stack(c, 1)
    bits = np.stack([words & np.uint64(0xffff), words >> np.uint64(16)], 2).reshape(-1)[:n - first]
    return torch.from_numpy((bits >= np.uint64(round(p * 65536))).copy()).cuda()


# ----------------------------------------------------------------------------------------------- together, streams, graphs
class Block:
    """A pre-norm residual block as a program would write it."""

    def __init__(self, seed, dim, hidden, t, grad=True):
        g = gen(seed)
        self.w, self.b = normal(g, dim, mean=1.0, scale=0.1), normal(g, dim, scale=0.1)
        self.gate, self.up = normal(g, hidden, dim, t=t, scale=dim ** -0.5), normal(g, hidden, dim, t=t, scale=dim ** -0.5)
        self.down = normal(g, dim, hidden, t=t, scale=hidden ** -0.5)
        self.params = [self.w, self.b, self.gate, self.up, self.down]
        for p in self.params:
            p.requires_grad_(grad)

    def __call__(self, x, rng, p=0.1, call=0):
        from muzero_amd import blocks
        h = blocks.gated_ff(blocks.layer_norm(x, self.w, self.b), self.gate, self.up)
        return blocks.dropout(torch.nn.functional.linear(h, self.down), p, rng, call, residual=x)

    def reference(self, x, keep, p=0.1):
        w, b, gate, up, down = (q.detach().double().requires_grad_() for q in self.params)
        xd = x.detach().double().requires_grad_()
        n = torch.nn.functional.layer_norm(xd, (xd.shape[-1],), w, b)
        h = torch.nn.functional.silu(n @ gate.t()) * (n @ up.t())
        y = xd + torch.where(keep, h @ down.t() * (65536 / (65536 - round(p * 65536))), 0.0)
        return y, [xd, w, b, gate, up, down]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [1, 144, 1000])
def test_block_of_all_three(rows, t):
    """layer_norm -> gated_ff -> linear -> dropout + residual, forward and gradients, against float64.  Four roundings to
    the type lie between input and output and seven between output gradient and a weight's gradient, each half(t) relative to
    its tensor's size; in norm they add up to no more than their sum (the products of the block keep norms to a
    factor of 2 at this scaling)."""
    t = TYPES[t]
    block = Block(1, 64, 160, t)
    x = normal(gen(2), rows, 64, t=t).requires_grad_()
    dy = normal(gen(3), rows, 64, t=t)
    rng = torch.tensor([5, 6], dtype=torch.int64, device="cuda")
    y = block(x, rng, call=2)
    got = [y.detach()] + list(torch.autograd.grad(y, [x] + block.params, dy))
    yr, wrt = block.reference(x, keep_mask(5, 6, 2, rows * 64, 0.1).view(rows, 64))
    want = [yr.detach()] + list(torch.autograd.grad(yr, wrt, dy.double()))
    for v, r, name in zip(got, want, ("y", "x", "w", "b", "gate", "up", "down")):
        off = (v.double() - r).norm() / r.norm()
        assert off <= 2 * 7 * max(half(t), 64 * U), (name, off.item())


@pytest.mark.parametrize("t", ["f32"])
def test_gradients_against_differences(t):
    """The directional derivative of the whole block by central differences in float64 of the reference, and of the
    kernels' own float32 forward pass, agree with the gradients."""
    block = Block(4, 48, 56, torch.float32)
    x = normal(gen(5), 70, 48).requires_grad_()
    dy = normal(gen(6), 70, 48)
    rng = torch.tensor([7, 8], dtype=torch.int64, device="cuda")
    leaves = [x] + block.params
    grads = torch.autograd.grad(block(x, rng), leaves, dy)
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        v = normal(gen(20 + i), *leaf.shape)
        v = v * (leaf.detach().norm() / v.norm())
        slope = (grad.double() * v.double()).sum().item()
        eps = 2.0 ** -8
        with torch.no_grad():
            kept = leaf.clone()
            f = []
            for sign in (1.0, -1.0):
                leaf.copy_(kept + sign * eps * v)
                f.append((block(x, rng).double() * dy.double()).sum().item())
            leaf.copy_(kept)
        size = grad.double().norm().item() * v.double().norm().item()
        # third-order term eps^2 (a few percent of size at most), rounding of f: u times the sum's size over 2 eps
        room = 4 * eps ** 2 * size + 64 * U * dy.double().norm().item() * 200 / (2 * eps)
        assert abs((f[0] - f[1]) / (2 * eps) - slope) <= room, (i, (f[0] - f[1]) / (2 * eps), slope, room)


def test_repeatable_and_on_another_stream():
    """The same bits on every run, also on a stream other than the default one while that one works on the same operands."""
    block = Block(9, 256, 512, torch.bfloat16)
    x = normal(gen(10), 3000, 256, t=torch.bfloat16).requires_grad_()
    dy = normal(gen(11), 3000, 256, t=torch.bfloat16)
    rng = torch.tensor([7, 8], dtype=torch.int64, device="cuda")

    def step():
        y = block(x, rng)
        return [y.detach()] + list(torch.autograd.grad(y, [x] + block.params, dy))

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            there = step()
        here = step()
        torch.cuda.synchronize()
        for a, b, c in zip(want, there, here):
            assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("rows", [16, 700])
def test_captured_training_steps(rows):
    """Forward and backward of the block recorded into two HIP graphs (other inputs, both alive), replayed in turn with
    new inputs, a new dropout state and eager work between the replays: every replay equals the eager step."""
    t = torch.bfloat16
    block = Block(12, 64, 136, t)
    graphs = []

    def step(x, dy, rng):
        leaf = x.detach().requires_grad_()
        y = block(leaf, rng)
        return [y.detach()] + list(torch.autograd.grad(y, [leaf] + block.params, dy))

    for k in range(2):
        x, dy = normal(gen(30 + k), rows, 64, t=t), normal(gen(40 + k), rows, 64, t=t)
        rng = torch.tensor([50 + k, 0], dtype=torch.int64, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, dy, rng)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(x, dy, rng)
        graphs.append((graph, x, dy, rng, outs))
    masks = set()
    for i in range(4):
        for graph, x, dy, rng, outs in graphs:
            x.copy_(normal(gen(100 + i), rows, 64, t=t))
            rng[1] += 1
            graph.replay()
        torch.cuda.synchronize()
        for graph, x, dy, rng, outs in graphs:
            for a, b in zip(outs, step(x, dy, rng)):
                assert torch.equal(a, b)
            masks.add(float(outs[0].double().sum()))
        torch.cuda.synchronize()
    assert len(masks) == 8


# ------------------------------------------------------------------------------------------- calls that programs also make
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,k,f", [(4483, 37, 509), (14100, 72, 257), (33000, 20, 130)])
def test_gated_ff_more_tiles_than_workgroups(rows, k, f, t):
    """Pair products of more tiles than the chip holds workgroups (they stay for several), ragged in all three."""
    x, wg, wu, bg, bu, dh = ff_inputs(rows, rows, k, f, TYPES[t])
    check_gated_ff(x, wg, wu, bg, bu, dh, "gelu", ff_run(x, wg, wu, bg, bu, dh, "gelu"))


def test_operands_that_lie_negated_in_memory():
    """The imaginary part of a conjugate is a view whose elements count with the other sign."""
    from muzero_amd import blocks
    z = torch.complex(normal(gen(1), 40, 1), normal(gen(2), 40, 1)).conj()
    x = z.imag
    assert x.is_neg()
    wg, wu = normal(gen(3), 24, 1), normal(gen(4), 24, 1)
    assert torch.equal(blocks.gated_ff(x, wg, wu), blocks.gated_ff(x.clone().resolve_neg(), wg, wu))
    rng = torch.zeros(2, dtype=torch.int64, device="cuda")
    assert torch.equal(blocks.dropout(x, 0.0, rng), x.clone().resolve_neg())
    leaf = normal(gen(5), 40, 1).requires_grad_()
    got, = torch.autograd.grad(blocks.dropout(leaf, 0.0, rng), leaf, x)
    assert torch.equal(got, x.clone().resolve_neg())


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad

    from muzero_amd import blocks
    x, w = torch.ones(20, 8, device="cuda"), torch.ones(6, 8, device="cuda")
    rng = torch.zeros(2, dtype=torch.int64, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: blocks.layer_norm(dual), lambda: blocks.gated_ff(dual, w, w),
                     lambda: blocks.gated_ff(x, w, forward_ad.make_dual(w, w)), lambda: blocks.dropout(dual, 0.5, rng)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


def test_autocast_leaves_float64_alone():
    from muzero_amd import blocks
    x, w = torch.ones(20, 8, device="cuda"), torch.ones(6, 8, device="cuda", dtype=torch.float64)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with pytest.raises(ValueError, match="dtype"):
            blocks.gated_ff(x, w, w)


def test_recomputed_activations_draw_the_same_mask():
    """Under torch.utils.checkpoint the forward pass runs again during the backward pass: the same gradients."""
    from torch.utils.checkpoint import checkpoint
    block = Block(13, 64, 96, torch.float32)
    x = normal(gen(14), 200, 64).requires_grad_()
    dy = normal(gen(15), 200, 64)
    rng = torch.tensor([3, 1], dtype=torch.int64, device="cuda")
    want = torch.autograd.grad(block(x, rng, 0.5), [x] + block.params, dy)
    got = torch.autograd.grad(checkpoint(block, x, rng, 0.5, use_reentrant=False), [x] + block.params, dy)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_threads_at_once():
    """Two threads, each with its own stream and operands, train and infer at the same time: each gets its own results."""
    import threading
    work = []
    for i, rows in enumerate((300, 1100)):
        block = Block(60 + i, 96, 200, torch.bfloat16)
        x = normal(gen(70 + i), rows, 96, t=torch.bfloat16).requires_grad_()
        work.append((block, x, normal(gen(80 + i), rows, 96, t=torch.bfloat16), torch.tensor([i, 9], dtype=torch.int64, device="cuda")))

    def step(block, x, dy, rng):
        y = block(x, rng)
        return [y.detach()] + list(torch.autograd.grad(y, [x] + block.params, dy))

    want = [step(*w) for w in work]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i].append(step(*work[i]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for i in range(2):
        assert len(got[i]) == 10
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(want[i], outs))


def test_gate_and_up_may_be_one_matrix_and_outputs_may_be_summed_twice():
    """The same tensor in two places: gradients add up; a graph kept for a second backward pass gives the same again."""
    from muzero_amd import blocks
    x, w, _, b, _, dh = ff_inputs(90, 70, 40, 48, torch.float32)
    leaf, wl, bl = (v.detach().requires_grad_() for v in (x, w, b))
    h = blocks.gated_ff(leaf, wl, wl, bl, bl)
    first = torch.autograd.grad(h, (leaf, wl, bl), dh, retain_graph=True)
    again = torch.autograd.grad(h, (leaf, wl, bl), dh)
    parts = ff_run(x, w, w, b, b, dh, "silu")
    assert torch.equal(first[1], parts[2] + parts[3]) and torch.equal(first[2], parts[4] + parts[5])
    assert all(torch.equal(a, c) for a, c in zip(first, again))
    leaf = x.detach().requires_grad_()
    rng = torch.zeros(2, dtype=torch.int64, device="cuda")
    both = torch.autograd.grad(blocks.dropout(leaf, 0.25, rng, residual=leaf), leaf, x)[0]
    assert torch.equal(both, x + blocks.dropout(x, 0.25, rng))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [9, 150, 2300])
def test_gated_ff_large_biases(rows, t):
    """Biases far above the products: the definition's, in float32 to its last digits (the bias is added to the finished
    sum, whose own error it does not enter)."""
    t = TYPES[t]
    x, wg, wu, bg, bu, dh = ff_inputs(95, rows, 520, 72, t)
    bg, bu = (bg.float() * 400).to(t), (bu.float() * 400).to(t)
    if t == torch.float32:
        check_gated_ff(x, wg, wu, bg, bu, dh, "relu", ff_run(x, wg, wu, bg, bu, dh, "relu"))
    else:
        h = ff_run(x, wg, wu, bg, bu, dh, "relu")[0]
        gate, up = x.double() @ wg.double().t() + bg.double(), x.double() @ wu.double().t() + bu.double()
        # a sum that starts at the bias passes through at most K additions: K u (sum|terms| + |bias|) each
        e_g, e_u = (521 * U * (x.double().abs() @ w.double().abs().t() + b.double().abs()) for w, b in ((wg, bg), (wu, bu)))
        ref = gate.clamp(min=0) * up
        fits = ref.abs() < 0.99 * torch.finfo(t).max
        assert fits.float().mean() > 0.9
        within(h[fits], ref[fits], (e_g * up.abs() + gate.abs() * e_u + e_g * e_u + 3 * U * ref.abs())[fits], "h")


def test_transforms_that_see_only_torch_operations_are_refused():
    """A trace, a batched or a functional transform would not record the kernels: an error, never a wrong result."""
    from muzero_amd import blocks
    x, w = torch.ones(20, 8, device="cuda"), torch.ones(6, 8, device="cuda")
    rng = torch.zeros(2, dtype=torch.int64, device="cuda")
    calls = (lambda v: blocks.layer_norm(v), lambda v: blocks.gated_ff(v, w, w), lambda v: blocks.dropout(v, 0.5, rng))
    for call in calls:
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(call, (x,), check_trace=False)
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(x.expand(3, 20, 8))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: call(v).sum())(x)
        with pytest.raises(ValueError, match="without memory"):
            call(torch._efficientzerotensor((20, 8), device="cuda"))


def test_graphed_callables():
    """torch.cuda.make_graphed_callables: forward and backward as two graphs, several steps with other inputs."""
    from muzero_amd import blocks

    class Module(torch.nn.Module):
        def __init__(self):
            super().__init__()
            g = gen(21)
            self.w, self.b = torch.nn.Parameter(normal(g, 64, mean=1.0)), torch.nn.Parameter(normal(g, 64))
            self.gate, self.up = torch.nn.Parameter(normal(g, 96, 64)), torch.nn.Parameter(normal(g, 96, 64))

        def forward(self, x):
            return blocks.gated_ff(blocks.layer_norm(x, self.w, self.b), self.gate, self.up, activation="gelu")

    eager, module = Module(), Module()
    graphed = torch.cuda.make_graphed_callables(module, (normal(gen(22), 150, 64).requires_grad_(),))
    for i in range(3):
        x, dy = normal(gen(30 + i), 150, 64).requires_grad_(), normal(gen(40 + i), 150, 96)
        want = torch.autograd.grad(eager(x), [x] + list(eager.parameters()), dy)
        got = torch.autograd.grad(graphed(x), [x] + list(module.parameters()), dy)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
