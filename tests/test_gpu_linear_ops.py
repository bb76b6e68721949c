"""Dropout, the linear layer with its epilogue and the loss head without logits on the GPU, against
plain 64-bit forms (tests/linear_ops_ref.py). Tolerances count roundings: H16 and H32 are half a
step of bf16 and f32 relative to the value; a product of length K accumulated in f32 is off by at
most about K steps of the sum of its terms' magnitudes (ACC per term, two half steps: the tensor
cores may truncate)."""
import math
import os
import subprocess
import sys

import pytest

import linear_ops_ref as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
BF, F32 = torch.bfloat16, torch.float32
H16, H32 = 2.0 ** -8, 2.0 ** -24
ACC = 2.0 ** -23
# 2-norm of a gradient's error over its own: the roundings of the products' bf16 operand and of the
# bf16 result, each at most H16 with a root mean square of at most H16 / sqrt(3)
NORM16 = math.sqrt(2.0 / 3.0) * H16 * 1.1


def _mat(g, rows, cols, dtype, dev, scale=1.0, offset=0, pad=0, fill=float("nan")):
    """A [rows, cols] view with `fill` everywhere around it: behind each row, before and after."""
    ld = -(-(cols + pad) // 8) * 8 if offset % 8 == 0 and pad % 8 == 0 else cols + pad
    buf = torch.full((offset + rows * ld + 64,), fill, dtype=dtype, device=dev)
    v = buf[offset:offset + rows * ld].view(rows, ld)[:, :cols] if rows else \
        torch.empty(0, cols, dtype=dtype, device=dev)
    v.copy_((torch.randn(rows, cols, generator=g) * scale).to(dtype))
    return v, buf


def _guard(rows, cols, dtype, dev, ld, offset=0):
    """An output view in a buffer of sentinels, and a check that nothing else was written."""
    buf = torch.full((offset + rows * ld + 64,), 7.0, dtype=dtype, device=dev)
    view = buf[offset:offset + rows * ld].view(rows, ld)[:, :cols]

    def check():
        b = buf.clone()
        b[offset:offset + rows * ld].view(rows, ld)[:, :cols] = 7.0
        assert bool((b == 7.0).all()), "written outside the output"
    return view, check


def _rng(dev, seed=0x1234567890ABCDEF, offset=0xFFFFFFF0):
    return torch.tensor([seed, offset], dtype=torch.int64, device=dev)


def _close(got, want, tol, what=""):
    got, want = got.double().cpu(), want.double().cpu()
    assert bool(torch.isfinite(got).all()), what + ": not finite"
    bad = (got - want).abs() > tol.double().cpu() + 1e-30
    assert not bool(bad.any()), (what, int(bad.sum()), float((got - want).abs().max()))


def _norm_close(got, want, tol, what=""):
    n = float(want.double().norm())
    e = float((got.double().cpu() - want.double().cpu()).norm())
    assert e <= tol * n + 1e-30, (what, e / max(n, 1e-30), tol)


# ------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (2, 256), (257, 300), (5, 4099),
                                       (64, 1024)])
@pytest.mark.parametrize("xt", [BF, F32])
@pytest.mark.parametrize("ot", [BF, F32])
@pytest.mark.parametrize("p,resid,offset,pad", [(0.1, False, 0, 0), (0.5, True, 0, 8),
                                                (0.25, True, 3, 5), (0.0, True, 0, 0),
                                                (1.0, True, 0, 0)])
def test_dropout(cuda, rows, cols, xt, ot, p, resid, offset, pad):
    from llmgpu import ops
    g = torch.Generator().manual_seed(rows * 7 + cols)
    x, _ = _mat(g, rows, cols, xt, cuda, 1.0, offset, pad)
    r, _ = _mat(g, rows, cols, ot, cuda, 2.0, offset, pad) if resid else (None, None)
    rng = _rng(cuda)
    ld = cols + 11 if offset else -(-cols // 8) * 8
    out, check = _guard(rows, cols, ot, cuda, ld, offset)
    ops.dropout_fwd(x, p, rng, site=37, resid=r, out=out)
    keep, scale = ref.keep_mask(0x1234567890ABCDEF, 0xFFFFFFF0 + 37, rows, cols, p)
    want = torch.where(keep, x.double().cpu() * scale, 0.0)
    mag = want.abs()
    if resid:
        want = want + r.double().cpu()
        mag = mag + r.double().cpu().abs()
    # the scale, the product and the sum round in f32, the result in its type
    tol = 3 * H32 * mag * (1 + H16) + (H16 if ot == BF else 0.0) * want.abs()
    _close(out, want, tol, "dropout")
    check()
    again = ops.dropout_fwd(x, p, rng, site=37, resid=r, out_dtype=ot)
    assert torch.equal(again, out)  # the same map wherever it is written


def test_dropout_dropped_elements_give_zero_whatever_they_hold(cuda):
    from llmgpu import ops
    rng = _rng(cuda, 3, 4)
    keep, _ = ref.keep_mask(3, 4, 64, 96, 0.5)
    keep = keep.to(cuda)
    for bad in (float("nan"), float("inf"), torch.finfo(F32).min):
        for pad in (0, 1):  # both memory paths
            x = torch.ones(64, 96 + pad, device=cuda)[:, :96]
            x[~keep] = bad
            y = ops.dropout_fwd(x, 0.5, rng)
            assert torch.equal(y, torch.where(keep, 2.0, 0.0))


def test_dropout_in_place_and_backward_mask(cuda):
    """out may be x or resid; the backward's mask is the forward's, in any type and layout."""
    from llmgpu import ops
    g = torch.Generator().manual_seed(2)
    rng = _rng(cuda, 9, 1 << 40)
    x, _ = _mat(g, 130, 1021, F32, cuda)
    r, _ = _mat(g, 130, 1021, F32, cuda, 1.0, 3, 5)
    want = ops.dropout_fwd(x, 0.3, rng, site=2, resid=r)
    a = x.clone()
    ops.dropout_fwd(a, 0.3, rng, site=2, resid=r, out=a)
    b = r.clone()
    ops.dropout_fwd(x, 0.3, rng, site=2, resid=b, out=b)
    assert torch.equal(a, want) and torch.equal(b, want)
    ones = torch.ones(130, 1021, dtype=BF, device=cuda)
    dx = ops.dropout_bwd(ones, 0.3, rng, site=2, out_dtype=F32)
    y = ops.dropout_fwd(torch.ones(130, 1021, device=cuda), 0.3, rng, site=2)
    assert torch.equal(dx, y)
    assert not torch.equal(y, ops.dropout_fwd(torch.ones(130, 1021, device=cuda), 0.3, rng, site=3))


def test_dropout_offsets_past_32_bits(cuda):
    """Rows whose element offsets pass 2^31 and 2^32 bytes and elements."""
    from llmgpu import ops
    rows, ld, cols = 90, 50_000_000, 24
    buf = torch.zeros(rows * ld, dtype=BF, device=cuda)
    x = buf.view(rows, ld)[:, :cols]
    x.fill_(1.0)
    y = ops.dropout_fwd(x, 0.5, _rng(cuda, 1, 2))
    keep, _ = ref.keep_mask(1, 2, rows, cols, 0.5)
    assert torch.equal(y.cpu() > 0, keep)
    ops.dropout_fwd(x, 0.5, _rng(cuda, 1, 2), out=x)
    assert torch.equal(x.cpu() > 0, keep)


def test_dropout_empty(cuda):
    from llmgpu import ops
    assert ops.dropout_fwd(torch.empty(0, 8, device=cuda), 0.5, _rng(cuda)).shape == (0, 8)
    assert ops.dropout_fwd(torch.empty(8, 0, device=cuda), 0.5, _rng(cuda)).shape == (8, 0)


# ------------------------------------------------------------------------------------- linear
def _linear_case(dev, M, K, N, act, p, out, resid, bias, w_mn, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x, _ = _mat(g, M, K, BF, dev, 1.0, 0, pad)
    w, _ = _mat(g, K if w_mn else N, N if w_mn else K, BF, dev, 1.5 / math.sqrt(K), 8, pad)
    b = (torch.randn(N, generator=g) * 0.5).to(dev) if bias else None
    r = _mat(g, M, N, out, dev, 2.0, 1, 2)[0] if resid else None
    return g, x, w, b, r


def _linear_want(x, w, b, r, act, p, w_mn, rng, site):
    wd = w.double() if w_mn else w.double().t()
    xd = x.double()
    z = xd @ wd
    ez = (x.shape[1] + 4) * ACC * (xd.abs() @ wd.abs())
    if b is not None:
        z = z + b.double()
        ez = ez + H32 * (z.abs() + b.double().abs())
    y = ref.act(z, act)
    # an activation's slope is at most 1.13; its sigmoid is off by a few steps times its argument
    e = 1.13 * ez + (8 + 2 * ref.sigmoid_arg(z, act).abs()) * 2 * H32 * y.abs()
    if p > 0:
        keep, scale = ref.keep_mask(int(rng[0]), int(rng[1]) + site, *z.shape, p)
        keep = keep.to(z.device)
        y, e = torch.where(keep, y * scale, 0.0), torch.where(keep, e * scale, 0.0)
        e = e + 2 * H32 * y.abs()
    if r is not None:
        y = y + r.double()
        e = e + H32 * (y.abs() + r.double().abs())
    return z, ez, y, e


SHAPES = [(1, 8, 1), (1, 768, 2304), (2, 40, 7), (3, 16, 300), (7, 1024, 257), (8, 264, 64),
          (9, 72, 33), (64, 128, 512), (127, 200, 129), (130, 768, 96), (300, 765, 1021),
          (513, 64, 640), (16, 4100, 37), (17, 264, 48),
          # products split along K: x w^T, dy w, dy^T x
          (40, 2101, 130), (300, 2048, 64), (33, 72, 2304), (2500, 40, 77),
          # tiles of 128 and 256 columns and of CTA pairs, whole and ragged
          (2048, 768, 768), (2100, 1100, 1304), (2100, 1100, 1301), (8192, 128, 512)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("act,p,out,resid,bias,w_mn", [
    ("none", 0.0, BF, False, True, False), ("gelu", 0.0, BF, False, True, True),
    ("none", 0.1, F32, True, True, True), ("relu", 0.25, BF, True, False, False),
    ("silu", 0.0, F32, False, False, False), ("gelu", 0.5, F32, True, True, False)])
def test_linear_fwd(cuda, M, K, N, act, p, out, resid, bias, w_mn):
    from llmgpu import ops
    _, x, w, b, r = _linear_case(cuda, M, K, N, act, p, out, resid, bias, w_mn, M + K + N, 8)
    rng, site = _rng(cuda, 77, 5), 3
    z, ez, want, e = _linear_want(x, w, b, r, act, p, w_mn, rng, site)
    y, pre = ops.linear_fwd(x, w, b, act, p, rng, site, r, w_mn, out_dtype=out, save_pre=True)
    tol = e + (H16 if out == BF else 0.0) * (want.abs() + e)
    _close(y, want, tol, "y")
    _close(pre, z, ez + H16 * (z.abs() + ez), "pre")
    # into rows of any stride and alignment, nothing around them touched
    for ld, off in ((-(-N // 8) * 8 + 8, 0), (N + 3, 5)):
        o, check = _guard(M, N, out, cuda, ld, off)
        ops.linear_fwd(x, w, b, act, p, rng, site, r, w_mn, out=o)
        _close(o, want, tol, "y into a view")
        check()
    if resid:  # the residual updated in place
        o = r.clone()
        ops.linear_fwd(x, w, b, act, p, rng, site, o, w_mn, out=o)
        _close(o, want, tol, "y over its residual")
    ops.check_device(cuda)


def _linear_bwd_want(dy, x, w, pre, act, p, w_mn, rng, site):
    dz = dy.double()
    if p > 0:
        keep, scale = ref.keep_mask(int(rng[0]), int(rng[1]) + site, *dz.shape, p)
        keep = keep.to(dz.device)
        dz = torch.where(keep, dz * scale, 0.0)
    e = 4 * H32 * dz.abs()
    if act != "none":
        zd = pre.double()
        gr = ref.act_grad(zd, act)
        # h + z h (1 - h) c: each sigmoid off by a few steps times its argument
        h = torch.sigmoid(ref.sigmoid_arg(zd, act))
        mag = h * (1 + zd.abs() * (1.6 * (1 + 0.14 * zd ** 2) if act == "gelu" else 1.0))
        eg = (16 + 4 * ref.sigmoid_arg(zd, act).abs()) * 2 * H32 * mag if act != "relu" else 0.0
        e = dz.abs() * eg + e * gr.abs()
        dz = dz * gr
    xd = x.double()
    wd = w.double().t() if w_mn else w.double()  # [N, K]
    dx, dw = dz @ wd, dz.t() @ xd
    ex = (H16 * dz.abs() + e) @ wd.abs() + (dz.shape[1] + 4) * ACC * (dz.abs() @ wd.abs())
    ew = (H16 * dz.abs() + e).t() @ xd.abs() + (dz.shape[0] + 4) * ACC * (dz.abs().t() @ xd.abs())
    if w_mn:
        dw, ew = dw.t(), ew.t()
    db = dz.sum(0)
    eb = e.sum(0) + (dz.shape[0] + 4) * H32 * dz.abs().sum(0)
    return dx, ex, dw, ew, db, eb


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("act,p,dyt,w_mn", [("none", 0.0, BF, False), ("none", 0.0, F32, True),
                                            ("none", 0.2, BF, True), ("gelu", 0.0, BF, False),
                                            ("silu", 0.1, F32, True), ("relu", 0.5, BF, False)])
def test_linear_bwd(cuda, M, K, N, act, p, dyt, w_mn):
    from llmgpu import ops
    g, x, w, _, _ = _linear_case(cuda, M, K, N, act, p, dyt, False, False, w_mn, M + K + N, 8)
    rng, site = _rng(cuda, 5, 99), 8
    dy = _mat(g, M, N, dyt, cuda, 0.1, 0 if N % 2 else 1, 8 if N % 2 else 3)[0]
    pre = _mat(g, M, N, BF, cuda, 2.0)[0] if act != "none" else None
    dx, ex, dw, ew, db, eb = _linear_bwd_want(dy, x, w, pre, act, p, w_mn, rng, site)
    gx, gw, gb = ops.linear_bwd(dy, x, w, pre, act, p, rng, site, w_mn)
    _close(gx, dx, ex + H16 * (dx.abs() + ex), "dx")
    _close(gw, dw, ew + H16 * (dw.abs() + ew), "dw")
    _close(gb, db, eb, "dbias")
    if M * N >= 4096:
        _norm_close(gx, dx, NORM16, "dx")
        _norm_close(gw, dw, NORM16, "dw")
    # f32 gradients, added to what is there; rows of any stride
    wr, wc = (K, N) if w_mn else (N, K)
    ow, check = _guard(wr, wc, BF, cuda, -(-wc // 8) * 8 + 8)
    ops.linear_bwd(dy, x, w, pre, act, p, rng, site, w_mn, dw=ow)
    assert torch.equal(ow, gw)
    check()
    aw, check = _guard(wr, wc, F32, cuda, wc + 3, 1)
    aw.fill_(0.5)
    ab = torch.full((N,), 2.0, device=cuda)
    gx32, _, _ = ops.linear_bwd(dy, x, w, pre, act, p, rng, site, w_mn, dx_dtype=F32, dw=aw, dbias=ab,
                                accumulate=True)
    _close(gx32, dx, ex, "f32 dx")
    _close(aw, dw + 0.5, ew + H32 * (dw.abs() + 0.5 + ew), "accumulated dw")
    _close(ab, db + 2.0, eb + H32 * (db.abs() + 2.0 + eb), "accumulated dbias")
    check()
    # each gradient alone
    assert torch.equal(ops.linear_bwd(dy, x, w, pre, act, p, rng, site, w_mn, need_dw=False,
                                      need_dbias=False)[0], gx)
    assert torch.equal(ops.linear_bwd(dy, x, w, pre, act, p, rng, site, w_mn, need_dx=False,
                                      need_dbias=False)[1], gw)
    assert torch.equal(ops.linear_bwd(dy, x, w, pre, act, p, rng, site, w_mn, need_dx=False,
                                      need_dw=False)[2], gb)
    ops.check_device(cuda)


@pytest.mark.parametrize("M", [5, 70])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("dyt,pad", [(BF, 0), (F32, 0), (F32, 3)])
def test_linear_bwd_dropped_places_count_nothing(cuda, M, act, dyt, pad):
    """What the forward dropped has no gradient, whatever dy and pre hold there."""
    from llmgpu import ops
    g = torch.Generator().manual_seed(M)
    K, N = 40, 72
    x, w = _mat(g, M, K, BF, cuda)[0], _mat(g, N, K, BF, cuda)[0]
    dy, pre = _mat(g, M, N, dyt, cuda, 1.0, 0, pad)[0], _mat(g, M, N, BF, cuda, 1.0, 0, pad)[0]
    rng = _rng(cuda, 31, 7)
    keep, _ = ref.keep_mask(31, 7 + 2, M, N, 0.5)
    gone = ~keep.to(cuda)
    want = None
    for dv, zv in ((0.0, 0.0), (math.nan, 1.0), (math.inf, 1.0), (1.0, math.nan), (1.0, math.inf),
                   (1.0, -math.inf), (torch.finfo(dyt).min, torch.finfo(BF).min)):
        dy[gone], pre[gone] = dv, zv
        got = ops.linear_bwd(dy, x, w, pre, act, 0.5, rng, 2)
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (dv, zv)
    assert all(bool(torch.isfinite(v).all()) for v in want)


@pytest.mark.parametrize("M", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("K,N", [(256, 37), (130, 1021), (768, 640)])
@pytest.mark.parametrize("act,p,dyt,w_mn", [("none", 0.0, F32, False), ("none", 0.3, BF, True),
                                            ("gelu", 0.0, BF, False), ("silu", 0.2, F32, True),
                                            ("relu", 0.5, BF, True)])
def test_linear_bwd_of_few_rows_keeps_dz(cuda, monkeypatch, M, K, N, act, p, dyt, w_mn):
    """dw of up to 8 rows comes from dz as it is: no rounding to bf16 stands between."""
    from llmgpu import ops
    monkeypatch.setitem(globals(), "H16", 0.0)  # _linear_bwd_want's rounding of dz
    g, x, w, _, _ = _linear_case(cuda, M, K, N, act, p, dyt, False, False, w_mn, M + K + N, 8)
    rng, site = _rng(cuda, 5, 99), 8
    dy = _mat(g, M, N, dyt, cuda, 0.1)[0]
    pre = _mat(g, M, N, BF, cuda, 2.0)[0] if act != "none" else None
    _, _, dw, ew, _, _ = _linear_bwd_want(dy, x, w, pre, act, p, w_mn, rng, site)
    aw = torch.full(tuple(w.shape), 0.5, device=cuda)
    ops.linear_bwd(dy, x, w, pre, act, p, rng, site, w_mn, dw=aw, dbias=torch.zeros(N, device=cuda),
                   accumulate=True)
    _close(aw, dw + 0.5, ew + H32 * (dw.abs() + 0.5 + ew), "accumulated dw")
    alone = ops.linear_bwd(dy, x, w, pre, act, p, rng, site, w_mn, dw=torch.zeros_like(aw), need_dx=False,
                           need_dbias=False)[1]
    _close(alone, dw, ew, "dw alone")
    ops.check_device(cuda)


def test_linear_bwd_of_few_rows_far_out(cuda):
    """f32's largest values, infinities and NaN in dy of few rows reach dw as they are, each in its own
    place alone."""
    from llmgpu import ops
    x = torch.ones(3, 8, dtype=BF, device=cuda)
    w = torch.zeros(8, 8, dtype=BF, device=cuda)
    for w_mn in (False, True):
        for v in (3.3e38, -3.3e38, torch.finfo(F32).max, 1e-37, math.inf, -math.inf, math.nan):
            dy = torch.zeros(3, 8, device=cuda)
            dy[1, 0] = v
            _, dw, _ = ops.linear_bwd(dy, x, w, w_mn=w_mn, dw=torch.zeros(8, 8, device=cuda))
            dw = dw if w_mn else dw.t()  # [K, N]
            assert torch.equal(dw[:, 0], dy[1, 0].expand(8)) or (math.isnan(v) and dw[:, 0].isnan().all())
            assert not dw[:, 1:].any()


@pytest.mark.parametrize("w_mn", [False, True])
def test_long_sums_in_f32(cuda, w_mn):
    """f32 results of operands that bf16 holds exactly: a chain is 32 accumulations of 16 products,
    each off by at most a step (2 H32) of the partial sum, however long the whole sum is."""
    from llmgpu import ops
    tol = 32 * 2 * H32
    for M, K, N in ((300, 16384, 520), (16384, 264, 520)):
        _, x, w, _, _ = _linear_case(cuda, M, K, N, "none", 0, F32, False, False, w_mn, M, 8)
        y, _ = ops.linear_fwd(x, w, w_mn=w_mn, out_dtype=F32)
        wd = w.double() if w_mn else w.double().t()
        _norm_close(y, x.double() @ wd, tol, "y")
        dy = torch.randn(M, N, device=cuda).to(BF)
        dw = torch.zeros(w.shape, device=cuda)
        dx, _, _ = ops.linear_bwd(dy, x, w, w_mn=w_mn, dx_dtype=F32, dw=dw)
        want = x.double().t() @ dy.double() if w_mn else dy.double().t() @ x.double()
        _norm_close(dw, want, tol, "dw")
        _norm_close(dx, dy.double() @ wd.t(), tol, "dx")
    ops.check_device(cuda)


def test_linear_no_rows(cuda):
    from llmgpu import ops
    x, w = torch.empty(0, 16, dtype=BF, device=cuda), torch.ones(24, 16, dtype=BF, device=cuda)
    y, _ = ops.linear_fwd(x, w)
    assert y.shape == (0, 24)
    dx, dw, db = ops.linear_bwd(y, x, w)
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    one = torch.ones(24, 16, device=cuda)
    ops.linear_bwd(y, x, w, dw=one, dbias=torch.ones(24, device=cuda), accumulate=True)
    assert bool((one == 1).all())


def test_linear_activations_at_the_ends(cuda):
    """Pre-activations of the type's largest values, infinities and NaN: relu, gelu and silu go
    to 0 on the left and to z on the right; their gradients at +-1e4 are 0 and 1."""
    from llmgpu import ops
    z = torch.tensor([-3e38, -1e20, -100.0, -0.0, 0.0, 100.0, 1e20, 3e38], device=cuda)
    x = torch.zeros(4, 8, dtype=BF, device=cuda)
    w = torch.zeros(8, 8, dtype=BF, device=cuda)
    for act in ("relu", "gelu", "silu"):
        y, _ = ops.linear_fwd(x, w, z, act, out_dtype=F32)
        assert torch.equal(y[0, 5:], z[5:]) and bool((y[0, :5].abs() <= 1e-30).all()), (act, y[0])
        pre = torch.tensor([-1e4, -100.0, 100.0, 1e4] * 2, device=cuda).to(BF).repeat(4, 1)
        dy = torch.ones(4, 8, device=cuda)
        _, _, db = ops.linear_bwd(dy, x, w, pre, act, need_dx=False, need_dw=False)
        assert torch.equal(db, torch.tensor([0.0, 0.0, 4.0, 4.0] * 2, device=cuda)), (act, db)
        nan, _ = ops.linear_fwd(x, w, torch.full((8,), float("nan"), device=cuda), act)
        assert bool(nan.isnan().all())


@pytest.mark.parametrize("M,N,K", [(64, 8192, 4800), (200, 1000, 4800), (2000, 64, 700), (40, 24, 64)])
def test_linear_bwd_products_beside_each_other(cuda, M, N, K):
    """dw's product may start beside dx's, and dx's beside the bias sum: what reads a gradient right
    after the call finds it whole, and what the call read may be overwritten. dy doubles from call
    to call, which doubles every gradient exactly."""
    from llmgpu import ops
    g = torch.Generator().manual_seed(M + N)
    x, _ = _mat(g, M, K, BF, cuda, 1.0, 0, 8)
    w, _ = _mat(g, N, K, BF, cuda, 1.0, 0, 8)
    v, _ = _mat(g, 24, K, BF, cuda, 1.0, 0, 8)
    base = torch.randn(M, N, generator=g).to(cuda)
    dy = base.clone()
    xs = torch.empty_strided(x.shape, x.stride(), dtype=BF, device=cuda)  # x's rows on 16 bytes

    def step(dx_dtype):
        dx, dw, db = ops.linear_bwd(dy, xs, w, dx_dtype=dx_dtype)
        xs.zero_()
        dy.zero_()
        read = [dx.clone(), dw.clone(), db.clone()]
        if dx_dtype == BF:
            read.append(ops.linear_fwd(dx, v)[0])
        return read

    for dtype in (BF, F32):
        dy.copy_(base), xs.copy_(x)
        first = step(dtype)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step(dtype)
        for i in range(1, 9):
            dy.copy_(base * 2.0 ** i), xs.copy_(x)
            got = step(dtype)
            assert all(torch.equal(a, b * 2.0 ** i) for a, b in zip(got, first)), (dtype, i)
            dy.copy_(base * 2.0 ** -i), xs.copy_(x)
            graph.replay()
            assert all(torch.equal(a, b * 2.0 ** -i) for a, b in zip(held, first)), (dtype, -i)
    ops.check_device(cuda)


def test_linear_gradients_far_out(cuda):
    """Pre-activations whose square or cube is past f32: the derivatives are 0 on the left and 1 on
    the right, and NaN stays NaN."""
    from llmgpu import ops
    z = torch.tensor([-1e36, -1e20, -1e13, -12.5, 12.5, 1e13, 1e20, 1e36], device=cuda)
    x, w = torch.zeros(4, 8, dtype=BF, device=cuda), torch.zeros(8, 8, dtype=BF, device=cuda)
    dy = torch.ones(4, 8, device=cuda)
    for act in ("relu", "gelu", "silu"):
        _, _, db = ops.linear_bwd(dy, x, w, z.to(BF).repeat(4, 1), act, need_dx=False, need_dw=False)
        # silu at +-12.5: e^-12.5 (1 + 12.5) = 5e-5 from its end; four rows are added up
        want = torch.tensor([0.0] * 4 + [4.0] * 4, dtype=torch.float64)
        at = torch.tensor([0.0] * 3 + [4 * 5.1e-5] * 2 + [0.0] * 3, dtype=torch.float64)
        assert bool(((db.double().cpu() - want).abs() <= at * (act == "silu")).all()), (act, db)
        if act != "relu":
            nan = torch.full((4, 8), float("nan"), dtype=BF, device=cuda)
            _, _, db = ops.linear_bwd(dy, x, w, nan, act, need_dx=False, need_dw=False)
            assert bool(db.isnan().all())


def test_linear_gradients_at_the_types_ends(cuda):
    """Pre-activations up to bf16's largest values: the derivatives are 0 on the left and 1 on the
    right (gelu's second term has a factor 2^-205 or less from |z| = 12 on)."""
    from llmgpu import ops
    top = torch.finfo(BF).max
    z = torch.tensor([-top, -3e38, -1.1e37, -1e37, 1e37, 1.1e37, 3e38, top], device=cuda).to(BF)
    x, w = torch.zeros(4, 8, dtype=BF, device=cuda), torch.zeros(8, 8, dtype=BF, device=cuda)
    dy = torch.ones(4, 8, device=cuda)
    want = torch.tensor([0.0] * 4 + [4.0] * 4, device=cuda)
    for act in ("relu", "gelu", "silu"):
        _, _, db = ops.linear_bwd(dy, x, w, z.repeat(4, 1), act, need_dx=False, need_dw=False)
        assert torch.equal(db, want), (act, db)
    # what overflowed to an infinity has gelu's limits
    inf = torch.tensor([-math.inf] * 4 + [math.inf] * 4, device=cuda).to(BF)
    _, _, db = ops.linear_bwd(dy, x, w, inf.repeat(4, 1), "gelu", need_dx=False, need_dw=False)
    assert torch.equal(db, want), db


# --------------------------------------------------------------------------------------- head
def _head_case(dev, rows, C, V, w_mn, ignored, seed, sharp=3.0):
    g = torch.Generator().manual_seed(seed)
    x, _ = _mat(g, rows, C, BF, dev, 1.0, 0, 8)
    w, _ = _mat(g, C if w_mn else V, V if w_mn else C, BF, dev, sharp / math.sqrt(C), 8, 8)
    t = torch.randint(0, V, (rows,), generator=g, dtype=torch.int32)
    if ignored:
        t[torch.rand(rows, generator=g) < 0.3] = -1
        t[rows // 2] = V  # past the vocabulary: left out too
    d = torch.rand(rows, generator=g) + 0.5
    return x, w, t.to(dev), d.to(dev)


def _head_want(x, w, t, d, scale, smoothing, w_mn):
    xd, wd = x.double(), w.double()
    if w_mn:
        wd = wd.t()
    loss, lse, z, y, valid = ref.head(xd, wd, t, smoothing)
    V, C = wd.shape
    ez = (C + 4) * ACC * (xd.abs() @ wd.abs().t())
    el = ez.amax(1) + (4 * H32) * (1 + lse.abs()) + 16 * H32
    # smoothing adds V terms of size smoothing / (V - 1): lse - z, each off by ez + el, summed in f32
    eloss = 2 * el + ez.amax(1) + 4 * H32 * loss.abs() + \
        smoothing * 4 * H32 * (lse.abs() + z.abs().amax(1)) * (1 + math.log2(V))
    coef = torch.where(valid, d.double() * scale, 0.0)[:, None]
    p = (z - lse[:, None]).exp()
    gr = coef * (p - y)
    eg = coef.abs() * (p * (ez + el[:, None] + (z - lse[:, None]).abs() * 4 * H32 + 8 * H32) +
                       4 * H32 * (p + y)) + H16 * gr.abs()
    dx, dw = gr @ wd, gr.t() @ xd
    ex = eg @ wd.abs() + (V + 4) * ACC * (gr.abs() @ wd.abs())
    ew = eg.t() @ xd.abs() + (xd.shape[0] + 4) * ACC * (gr.abs().t() @ xd.abs())
    if w_mn:
        dw, ew = dw.t(), ew.t()
    return loss, eloss, lse, el, dx, ex, dw, ew


HEADS = [(1, 64, 1, 0), (1, 768, 5003, 0), (5, 8, 100, 256), (33, 72, 257, 256), (256, 128, 256, 0),
         (130, 200, 1000, 512), (300, 765, 3001, 1024), (513, 264, 2048, 2048), (64, 64, 20011, 0),
         (1030, 768, 5003, 2560), (2048, 1024, 8192, 0)]


@pytest.mark.parametrize("rows,C,V,piece", HEADS)
@pytest.mark.parametrize("smoothing,w_mn,ignored", [(0.0, False, False), (0.1, True, True),
                                                    (0.0, True, False), (0.2, False, True)])
def test_loss_head(cuda, rows, C, V, piece, smoothing, w_mn, ignored):
    from llmgpu import ops
    x, w, t, d = _head_case(cuda, rows, C, V, w_mn, ignored, rows + C + V)
    loss, eloss, lse, el, dx, ex, dw, ew = _head_want(x, w, t, d, 0.5, smoothing, w_mn)
    gl, gs = ops.linear_cross_entropy_fwd(x, w, t, smoothing, w_mn)
    _close(gl, loss, eloss, "loss")
    _close(gs, lse, el, "lse")
    gx, gw = ops.linear_cross_entropy_bwd(x, w, t, gs, d, 0.5, smoothing, w_mn, piece=piece)
    _close(gx, dx, ex + H16 * (dx.abs() + ex), "dx")
    _close(gw, dw, ew + H16 * (dw.abs() + ew), "dw")
    left = (t < 0) | (t >= V)
    assert not bool(gl[left].any()) and not bool(gx[left].any())
    if rows * V >= 4096:
        _norm_close(gx, dx, NORM16, "dx")
        _norm_close(gw, dw, NORM16, "dw")
    wr, wc = (C, V) if w_mn else (V, C)
    ow, check = _guard(wr, wc, BF, cuda, -(-wc // 8) * 8 + 8)
    ops.linear_cross_entropy_bwd(x, w, t, gs, d, 0.5, smoothing, w_mn, dw=ow, piece=piece)
    assert torch.equal(ow, gw)
    check()
    aw, check = _guard(wr, wc, F32, cuda, wc + 3, 1)
    aw.fill_(0.25)
    gx32, _ = ops.linear_cross_entropy_bwd(x, w, t, gs, d, 0.5, smoothing, w_mn, dx_dtype=F32, dw=aw,
                                           accumulate=True, piece=piece)
    _close(gx32, dx, ex, "f32 dx")
    _close(aw, dw + 0.25, ew + H32 * (dw.abs() + 0.25 + ew), "accumulated dw")
    check()
    assert torch.equal(ops.linear_cross_entropy_bwd(x, w, t, gs, d, 0.5, smoothing, w_mn, piece=piece,
                                                    need_dw=False)[0], gx)
    assert torch.equal(ops.linear_cross_entropy_bwd(x, w, t, gs, d, 0.5, smoothing, w_mn, piece=piece,
                                                    need_dx=False)[1], gw)
    ops.check_device(cuda)


@pytest.mark.parametrize("rows,C,V,piece", [(256, 128, 256, 0), (300, 64, 2000, 512), (64, 4800, 600, 0)])
def test_loss_head_bwd_products_beside_each_other(cuda, rows, C, V, piece):
    """As for the linear layer: the weights of the rows double from call to call, and so do the
    gradients, exactly (the largest weight is divided out before the rounding)."""
    from llmgpu import ops
    x, w, t, d = _head_case(cuda, rows, C, V, False, False, 7)
    _, lse = ops.linear_cross_entropy_fwd(x, w, t)
    c, first = d.clone(), None
    for i in range(9):
        c.copy_(d * 2.0 ** i)
        dx, dw = ops.linear_cross_entropy_bwd(x, w, t, lse, c, piece=piece)
        c.zero_()
        got = [dx.clone(), dw.clone(), ops.linear_fwd(dx, w)[0]]
        first = first or got
        assert all(torch.equal(a, b * 2.0 ** i) for a, b in zip(got, first)), i
    ops.check_device(cuda)


def test_loss_head_of_one_class(cuda):
    """A vocabulary of one: the loss is 0 whatever the logit, smoothed or not, and so are its
    gradients, up to the rounding of lse (p = 2^(z log2 e - lse log2 e) with each term rounded)."""
    from llmgpu import ops
    for rows in (1, 40):
        x, w, t, d = _head_case(cuda, rows, 64, 1, False, False, 2)
        for s in (0.0, 0.1, 0.9):
            loss, lse = ops.linear_cross_entropy_fwd(x, w, t, s)
            dx, dw = ops.linear_cross_entropy_bwd(x, w, t, lse, d, 1.0, s, dx_dtype=F32)
            e = 8 * H32 * (1 + lse.double().abs()) * d.double()
            assert bool((loss.double().abs() <= e).all()), (s, loss)
            assert bool((dx.double().abs() <= e[:, None] * w.double().abs()).all()), (s, dx)
            assert bool((dw.double().abs() <= e @ x.double().abs() * (1 + H16)).all()), (s, dw)


def test_loss_head_rows_left_out_may_hold_anything(cuda):
    """A padded batch whose padding rows hold NaN and infinities: they reach nothing."""
    from llmgpu import ops
    x, w, t, d = _head_case(cuda, 70, 64, 700, False, True, 1)
    left = (t < 0) | (t >= 700)
    clean = [ops.linear_cross_entropy_fwd(x, w, t)]
    clean.append(ops.linear_cross_entropy_bwd(x, w, t, clean[0][1], d))
    for bad in (float("nan"), float("inf"), torch.finfo(BF).min):
        y = x.clone()
        y[left] = bad
        dd = d.clone()
        dd[left] = float("nan")
        loss, lse = ops.linear_cross_entropy_fwd(y, w, t)
        dx, dw = ops.linear_cross_entropy_bwd(y, w, t, lse, dd)
        assert torch.equal(loss, clean[0][0])
        assert torch.equal(dx, clean[1][0]) and torch.equal(dw, clean[1][1])
    none = torch.full_like(t, -1)  # every row left out
    loss, lse = ops.linear_cross_entropy_fwd(x, w, none)
    dx, dw = ops.linear_cross_entropy_bwd(x, w, none, lse, d)
    assert not loss.any() and not dx.any() and not dw.any()


def test_loss_head_extreme_logits(cuda):
    """Logits of -inf (a vocabulary entry ruled out) and rows of very large logits."""
    from llmgpu import ops
    C, V = 64, 300
    x = torch.zeros(40, C, dtype=BF, device=cuda)
    x[:, 0] = 1.0
    x[1::2, 0] = 1000.0
    g = torch.Generator().manual_seed(0)
    w = torch.zeros(V, C, dtype=BF)
    w[:, 0] = torch.randn(V, generator=g).to(BF)
    w[130:260, 0] = torch.finfo(BF).min  # -inf from the second row on, the lowest value in the first
    t = torch.randint(0, 130, (40,), generator=g, dtype=torch.int32).to(cuda)
    w = w.to(cuda)
    z = (x.float() @ w.float().t()).double()
    loss, lse = ops.linear_cross_entropy_fwd(x, w, t)
    want = torch.logsumexp(z, 1)
    _close(lse, want, 8 * H32 * (1 + want.abs()), "lse")
    wl = want - z.gather(1, t.long()[:, None])[:, 0]
    _close(loss, wl, 16 * H32 * (1 + want.abs()), "loss")
    dx, _ = ops.linear_cross_entropy_bwd(x, w[:130].contiguous(), t,
                                         ops.linear_cross_entropy_fwd(x, w[:130].contiguous(), t)[1])
    assert bool(torch.isfinite(dx.float()).all())


def test_loss_head_row_weights(cuda):
    """Weights of any kind: all zero; signs and sizes mixed over 60 binades; one that is infinite,
    which reaches its own row of dx (and dw) alone."""
    from llmgpu import ops
    x, w, t, _ = _head_case(cuda, 96, 64, 400, False, False, 8)
    _, lse = ops.linear_cross_entropy_fwd(x, w, t)
    dx, dw = ops.linear_cross_entropy_bwd(x, w, t, lse, torch.zeros(96, device=cuda))
    assert not dx.any() and not dw.any()
    g = torch.Generator().manual_seed(1)
    d = (torch.randn(96, generator=g) * torch.exp2(torch.randint(-30, 30, (96,), generator=g))).to(cuda)
    _, _, _, _, wx, ex, ww, ew = _head_want(x, w, t, d, 2.0, 0.0, False)
    dx, dw = ops.linear_cross_entropy_bwd(x, w, t, lse, d, 2.0)
    _close(dx, wx, ex + H16 * (wx.abs() + ex), "dx")
    _close(dw, ww, ew + H16 * (ww.abs() + ew), "dw")
    one = torch.ones(96, device=cuda)
    dx, _ = ops.linear_cross_entropy_bwd(x, w, t, lse, one)
    one[17] = float("inf")
    ix, _ = ops.linear_cross_entropy_bwd(x, w, t, lse, one)
    keep = torch.arange(96, device=cuda) != 17
    assert torch.equal(ix[keep], dx[keep]) and not bool(torch.isfinite(ix[17].float()).all())


def test_loss_head_no_rows(cuda):
    from llmgpu import ops
    x, w = torch.empty(0, 16, dtype=BF, device=cuda), torch.ones(40, 16, dtype=BF, device=cuda)
    t = torch.empty(0, dtype=torch.int32, device=cuda)
    loss, lse = ops.linear_cross_entropy_fwd(x, w, t)
    dx, dw = ops.linear_cross_entropy_bwd(x, w, t, lse)
    assert loss.shape == (0,) and dx.shape == (0, 16) and not dw.any()


def test_loss_head_agrees_with_cross_entropy_over_logits(cuda):
    """The framework's loss over logits in memory, on the same (bf16-rounded) logits: an identity
    weight makes the head's logits the rows of x themselves. The gradients agree with smoothed
    labels too; the loss over logits leaves the smoothing out of what it reports."""
    from llmgpu import ops
    g = torch.Generator().manual_seed(4)
    V = 512
    x = (torch.randn(96, V, generator=g) * 2).to(BF).to(cuda)
    w = torch.eye(V, dtype=BF, device=cuda)
    t = torch.randint(0, V, (96,), generator=g, dtype=torch.int32).to(cuda)
    logits = x.clone()
    want = ops.cross_entropy(logits, V, t, 0.5, 0.1)
    loss, lse = ops.linear_cross_entropy_fwd(x, w, t)
    assert float((loss - want).abs().max()) < 2e-5  # f32 sums of 512 terms on both sides
    dx, _ = ops.linear_cross_entropy_bwd(x, w, t, lse, None, 0.5, 0.1)
    # both round the same gradient to bf16 (dx = G I exactly); a difference in the last f32 bits
    # can cross a rounding border: one step
    assert float((dx.float() - logits.float()).abs().max()) <= 2 * H16 * float(logits.float().abs().max())


# -------------------------------------------------------------------------- gradients by difference
def test_gradients_against_differences(cuda):
    """Central differences of the operators' own forward along directions that bf16 holds exactly:
    inputs are multiples of 1/16 below 4, the step is 1/16, so x +- h d are exact. The cubic
    term of a difference is at most h^2 / 6 times the third derivative along d."""
    from llmgpu import ops
    g = torch.Generator().manual_seed(12)
    rows, C, V, h = 24, 32, 96, 1.0 / 16

    def grid(*shape):
        return (torch.randint(-16, 17, shape, generator=g) / 16).to(BF).to(cuda)
    x, w = grid(rows, C), grid(V, C)
    t = torch.randint(0, V, (rows,), generator=g, dtype=torch.int32).to(cuda)

    def loss(a, b):
        return ops.linear_cross_entropy_fwd(a, b, t, 0.1)[0].double().sum().item()
    _, lse = ops.linear_cross_entropy_fwd(x, w, t, 0.1)
    dx, dw = ops.linear_cross_entropy_bwd(x, w, t, lse, None, 1.0, 0.1)
    for grad, at in ((dx, 0), (dw, 1)):
        for _ in range(4):
            # one coordinate per row of x (rows do not interact) or a single entry of w
            d = torch.zeros_like(x if at == 0 else w)
            if at == 0:
                d[torch.arange(rows), torch.randint(0, C, (rows,), generator=g)] = 1.0
            else:
                d[int(torch.randint(0, V, (1,), generator=g)), int(torch.randint(0, C, (1,), generator=g))] = 1.0
            hi = (x + h * d, w) if at == 0 else (x, w + h * d)
            lo = (x - h * d, w) if at == 0 else (x, w - h * d)
            got = (loss(*hi) - loss(*lo)) / (2 * h)
            want = float((grad.double() * d.double()).sum())
            # |third derivative| of a log-sum-exp along a unit coordinate: at most 2 max |c|^3 per
            # row, |c| <= 1 (its coefficients are entries of x or w, at most 1)
            tol = rows * (2 * h * h / 6) + 2 * H16 * float((grad.double() * d.double()).abs().sum()) + \
                rows * 64 * H32 / h
            assert abs(got - want) <= tol, (at, got, want, tol)
    # the linear layer: silu, dropout, bias; the sum of its f32 outputs weighted by dy
    xl, wl = grid(rows, C), grid(48, C)
    b = torch.zeros(48, device=cuda)
    rng = _rng(cuda, 6, 7)
    dy = torch.randn(rows, 48, generator=g).to(cuda)

    def total(a, m, c):
        y, _ = ops.linear_fwd(a, m, c, "silu", 0.25, rng, 1, out_dtype=F32)
        return (y.double() * dy.double()).sum().item()
    _, pre = ops.linear_fwd(xl, wl, b, "silu", 0.25, rng, 1, save_pre=True)
    gx, gw, gb = ops.linear_bwd(dy, xl, wl, pre, "silu", 0.25, rng, 1)
    for grad, at in ((gx, 0), (gw, 1), (gb, 2)):
        for k in range(4):
            args_hi, args_lo = [xl, wl, b], [xl, wl, b]
            d = torch.zeros_like(args_hi[at])
            d.view(-1)[int(torch.randint(0, d.numel(), (1,), generator=g))] = 1.0
            args_hi[at], args_lo[at] = args_hi[at] + h * d, args_lo[at] - h * d
            got = (total(*args_hi) - total(*args_lo)) / (2 * h)
            want = float((grad.double() * d.double()).sum())
            # silu''' is below 0.6; pre is rounded to bf16 (|z| below 16: off by 16 H16, silu'' below
            # 0.5); dz and the gradient are rounded to bf16
            reach = float(dy.double().abs().sum()) / 0.75 / (1 if at == 0 else 48) * 4
            tol = reach * (0.6 * h * h / 6 + 8 * H16 + 2 * H16 + 64 * H32 / h)
            assert abs(got - want) <= tol, (at, got, want, tol)


# ------------------------------------------------------------------------------ large matrices
def test_linear_offsets_past_32_bits(cuda):
    """Results and gradients of more than 2^31 elements: rows on both sides of the border."""
    from llmgpu import ops
    M, K, N = 70000, 64, 32768
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(M, K, generator=g, device=cuda).to(BF)
    w = (torch.randn(N, K, generator=g, device=cuda) * 0.2).to(BF)
    rng = _rng(cuda, 8, 9)
    rows = torch.tensor([0, 1, 40000, 65535, 65536, 65537, M - 1])
    keep, scale = _rows_mask(8, 9, rows, N, 0.25)
    keep = keep.to(cuda)
    y, pre = ops.linear_fwd(x, w, None, "gelu", 0.25, rng, save_pre=True)
    rows = rows.to(cuda)
    z, ez, _, _ = _linear_want(x[rows], w, None, None, "gelu", 0.0, False, rng, 0)
    want = torch.where(keep, ref.act(z, "gelu") * scale, 0.0)
    tol = scale * (1.13 * ez + (8 + 2 * ref.sigmoid_arg(z, "gelu").abs()) * 2 * H32 *
                   ref.act(z, "gelu").abs()) + (H16 + 2 * H32) * want.abs()
    _close(y[rows], want, tol, "y")
    _close(pre[rows], z, ez + H16 * (z.abs() + ez), "pre")
    dy = y  # any matrix of that size
    dx, dw, db = ops.linear_bwd(dy, x, w, pre, "gelu", 0.25, rng)
    dz = torch.where(keep, dy[rows].double() * scale, 0.0) * ref.act_grad(pre[rows].double(), "gelu")
    _norm_close(dx[rows], dz @ w.double(), NORM16, "dx")
    # dw and dbias over all rows, in 64 bits on the device
    n0, n1 = 17, 33
    keep_n = _rows_mask(8, 9, torch.arange(M), n1, 0.25)[0][:, n0:n1].to(cuda)
    zc = pre[:, n0:n1].double()
    dzc = torch.where(keep_n, dy[:, n0:n1].double() * scale, 0.0) * ref.act_grad(zc, "gelu")
    _norm_close(dw[n0:n1], dzc.t() @ x.double(), NORM16, "dw")
    _norm_close(db[n0:n1], dzc.sum(0), 1e-5, "dbias")
    ops.check_device(cuda)


def _rows_mask(seed, offset, rows, cols, p):
    """ref.keep_mask for some rows of a matrix."""
    import numpy as np
    n8 = (cols + 7) // 8
    one = np.ones((len(rows), n8), dtype=np.uint64)
    words = ref.philox([one * np.arange(n8, dtype=np.uint64), one * rows.numpy().astype(np.uint64)[:, None],
                        one * np.uint64(offset), one * np.uint64(0)], (seed, 0))
    lanes = np.stack([(v >> np.uint64(16 * h)) & np.uint64(0xFFFF) for v in words for h in (0, 1)], -1)
    t = round(p * 65536)
    keep = lanes.reshape(len(rows), n8 * 8)[:, :cols].astype(np.int64) >= t
    return torch.from_numpy(keep), 65536 / (65536 - t)


def test_loss_head_of_many_rows(cuda):
    """70000 rows by 33000 classes: 2.3e9 logits, in pieces of the library's choice."""
    from llmgpu import ops
    rows, C, V = 70000, 64, 33000
    g = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn(rows, C, generator=g, device=cuda).to(BF)
    w = (torch.randn(V, C, generator=g, device=cuda) * 0.4).to(BF)
    t = torch.randint(-1, V, (rows,), generator=g, device=cuda, dtype=torch.int32)
    d = torch.rand(rows, generator=g, device=cuda) / rows
    loss, lse = ops.linear_cross_entropy_fwd(x, w, t)
    dx, dw = ops.linear_cross_entropy_bwd(x, w, t, lse, d)
    wd = w.double()
    want_dw = torch.zeros(V, C, dtype=torch.float64, device=cuda)
    for r in range(0, rows, 2000):
        s = slice(r, r + 2000)
        ls, le, z, y, valid = ref.head(x[s].double(), wd, t[s], 0.0)
        # sums of 33000 exponentials in f32, each slot of 128 merged in turn; logits of 64 products
        assert float((loss[s].double() - ls).abs().max()) < 2e-5
        assert float((lse[s].double() - le).abs().max()) < 2e-5
        gr = torch.where(valid, d[s].double(), 0.0)[:, None] * ((z - le[:, None]).exp() - y)
        _norm_close(dx[s], gr @ wd, NORM16, "dx")
        want_dw += gr.t() @ x[s].double()
    _norm_close(dw, want_dw, NORM16, "dw")
    ops.check_device(cuda)


# ----------------------------------------------------------------------------- used together
def _block(ops, s, rng):
    """Embedding dropout, a feed-forward block with its residual, the head's loss, and the way back:
    the losses and every gradient."""
    x0 = ops.dropout_fwd(s["x"], 0.1, rng, site=0)
    a, pre = ops.linear_fwd(x0, s["w1"], s["b1"], "gelu", save_pre=True)
    y, _ = ops.linear_fwd(a, s["w2"], s["b2"], "none", 0.1, rng, 1, resid=x0, w_mn=True)
    loss, lse = ops.linear_cross_entropy_fwd(y, s["wv"], s["t"])
    dy, dwv = ops.linear_cross_entropy_bwd(y, s["wv"], s["t"], lse, s["d"])
    da, dw2, db2 = ops.linear_bwd(dy, a, s["w2"], None, "none", 0.1, rng, 1, w_mn=True)
    dx0, dw1, db1 = ops.linear_bwd(da, x0, s["w1"], pre, "gelu")
    dx = ops.dropout_bwd(dx0 + dy, 0.1, rng, site=0)
    return dict(loss=loss, dwv=dwv, dw2=dw2, db2=db2, dw1=dw1, db1=db1, dx=dx)


def _block_state(cuda, seed, rows=200, C=96, F=256, V=517):
    g = torch.Generator().manual_seed(seed)

    def m(r, c, scale):
        return _mat(g, r, c, BF, cuda, scale)[0]
    return dict(x=m(rows, C, 1.0), w1=m(F, C, 0.1), w2=m(F, C, 0.06), wv=m(V, C, 0.2),
                b1=(torch.randn(F, generator=g) * 0.1).to(cuda),
                b2=(torch.randn(C, generator=g) * 0.1).to(cuda),
                t=torch.randint(-1, V, (rows,), generator=g, dtype=torch.int32).to(cuda),
                d=torch.full((rows,), 1.0 / rows, device=cuda))


def _block_want(s, rng):
    """The same in 64 bits by autograd."""
    v = {k: s[k].double().cpu().requires_grad_(True) for k in ("x", "w1", "w2", "wv", "b1", "b2")}
    rows, C = s["x"].shape
    seed, off = (int(q) for q in rng.tolist())
    k0, sc = ref.keep_mask(seed, off, rows, C, 0.1)
    k1, _ = ref.keep_mask(seed, off + 1, rows, C, 0.1)
    x0 = torch.where(k0, v["x"] * sc, 0.0)
    a = ref.act(x0 @ v["w1"].t() + v["b1"], "gelu")
    y = x0 + torch.where(k1, (a @ v["w2"] + v["b2"]) * sc, 0.0)
    loss = ref.head(y, v["wv"], s["t"].cpu(), 0.0)[0]
    (loss * s["d"].double().cpu()).sum().backward()
    return dict(loss=loss.detach(), dwv=v["wv"].grad, dw2=v["w2"].grad, db2=v["b2"].grad,
                dw1=v["w1"].grad, db1=v["b1"].grad, dx=v["x"].grad)


def test_block_forward_and_backward(cuda):
    """Every value passes at most 8 roundings to bf16 on its way (x0, pre, a, y, the gradients by
    logits, dy, dz twice), each with a root mean square of at most H16 / sqrt(3)."""
    from llmgpu import ops
    s, rng = _block_state(cuda, 3), _rng(cuda, 21, 4)
    got, want = _block(ops, s, rng), _block_want(s, rng)
    for k in want:
        _norm_close(got[k], want[k], 8 * H16 / math.sqrt(3), k)
    ops.check_device(cuda)


def test_block_is_repeatable_and_captures(cuda):
    """Same bits on every run and in a captured graph; a replay reads the generator's new offset;
    two graphs and eager calls on two streams do not disturb one another."""
    from llmgpu import ops
    s, s2 = _block_state(cuda, 3), _block_state(cuda, 4, rows=333, C=64, F=128, V=1000)
    rng, rng2 = _rng(cuda, 21, 4), _rng(cuda, 5, 6)
    first = _block(ops, s, rng)
    for k, v in _block(ops, s, rng).items():
        assert torch.equal(v, first[k]), k
    other = _block(ops, s2, rng2)
    torch.cuda.synchronize()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = _block(ops, s, rng)
    with torch.cuda.graph(g2):
        o2 = _block(ops, s2, rng2)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(a):
            g1.replay()
        with torch.cuda.stream(b):
            g2.replay()
    e = _block(ops, s, rng)
    torch.cuda.synchronize()
    for k in first:
        assert torch.equal(o1[k], first[k]) and torch.equal(e[k], first[k]), k
        assert torch.equal(o2[k], other[k]), k
    rng[1] += 1000
    g1.replay()
    torch.cuda.synchronize()
    moved = _block(ops, s, rng)
    assert all(torch.equal(o1[k], moved[k]) for k in moved)
    assert not torch.equal(moved["dx"], first["dx"])
    ops.check_device(cuda)


def test_two_calls_at_once(cuda):
    """The same operators at once on two streams, each with its own workspace."""
    from llmgpu import ops
    s = [_block_state(cuda, 10 + i, rows=700, C=128, F=512, V=3000) for i in range(2)]
    rng = _rng(cuda, 1, 1)
    want = [_block(ops, q, rng) for q in s]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = _block(ops, s[i], rng)
    torch.cuda.synchronize()
    for i in range(2):
        for k in want[i]:
            assert torch.equal(got[i][k], want[i][k]), (i, k)


def test_plain_c_calls_equal_the_wrappers(cuda):
    """Each C entry point called with its own argument list, on a stream of its own."""
    from llmgpu import load, ops
    lib = load()
    g = torch.Generator().manual_seed(5)
    M, K, N = 70, 96, 136
    x, w = _mat(g, M, K, BF, cuda)[0], _mat(g, N, K, BF, cuda, 0.1)[0]
    b = torch.randn(N, generator=g).to(cuda)
    r = torch.randn(M, N, generator=g).to(cuda)
    t = torch.randint(-1, N, (M,), generator=g, dtype=torch.int32).to(cuda)
    d = torch.rand(M, generator=g).to(cuda)
    rng = _rng(cuda, 3, 1 << 50)
    want = [ops.dropout_fwd(x, 0.3, rng, 2 ** 63 + 5)]
    want += ops.linear_fwd(x, w, b, "gelu", 0.2, rng, 7, r, out_dtype=F32, save_pre=True)
    want += ops.linear_bwd(r, x, w, want[2], "gelu", 0.2, rng, 7)
    want += ops.linear_cross_entropy_fwd(x, w, t, 0.1)
    want += ops.linear_cross_entropy_bwd(x, w, t, want[7], d, 3.0, 0.1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = [torch.zeros_like(v) for v in want]
    work = torch.empty(1 << 24, dtype=torch.uint8, device=cuda)
    torch.cuda.synchronize()
    st, ld = s.cuda_stream, x.stride(0)

    def p(v):
        return v.data_ptr()
    assert lib.llmgpu_op_dropout(p(x), 0, ld, None, 0, p(got[0]), 0, K, M, K, 0.3, p(rng), 2 ** 63 + 5,
                                 st) == 0
    assert lib.llmgpu_op_linear_fwd(p(x), ld, p(w), w.stride(0), 0, p(b), 2, 0.2, p(rng), 7, p(r), N,
                                    p(got[2]), N, p(got[1]), 1, N, M, N, K, p(work), None, st) == 0
    assert lib.llmgpu_op_linear_bwd(p(r), 1, N, p(x), ld, p(w), w.stride(0), 0, p(want[2]), N, 2, 0.2,
                                    p(rng), 7, p(got[3]), 0, K, p(got[4]), 0, K, p(got[5]), 0, M, N, K,
                                    p(work), None, st) == 0
    assert lib.llmgpu_op_linear_ce_fwd(p(x), ld, p(w), w.stride(0), 0, p(t), M, K, N, 0.1, p(got[6]),
                                       p(got[7]), p(work), None, st) == 0
    assert lib.llmgpu_op_linear_ce_bwd(p(x), ld, p(w), w.stride(0), 0, p(t), p(want[7]), p(d), 3.0, M, K,
                                       N, 0.1, p(got[8]), 0, K, p(got[9]), 0, K, 0, 0, p(work), None,
                                       st) == 0
    torch.cuda.synchronize()
    for i, (a, c) in enumerate(zip(got, want)):
        assert torch.equal(a, c), i


@pytest.mark.parametrize("M,K,N", [(256, 4096, 512), (40, 2101, 130), (2048, 768, 768)])
def test_plain_c_linear_forward_stays_in_its_workspace(cuda, M, K, N):
    """With a workspace of llmgpu_op_linear_fwd_work bytes (products split along K and others), and
    with none, which leaves K whole: the same to f32 rounding, nothing written behind it."""
    from llmgpu import load, ops
    lib = load()
    g = torch.Generator().manual_seed(K)
    x, w = _mat(g, M, K, BF, cuda)[0], _mat(g, N, K, BF, cuda, 1 / math.sqrt(K))[0]
    n = lib.llmgpu_op_linear_fwd_work(M, N, K)
    buf = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device=cuda)
    y, z = torch.empty(M, N, device=cuda), torch.empty(M, N, device=cuda)
    st = torch.cuda.current_stream().cuda_stream
    for out, work in ((y, buf.data_ptr()), (z, None)):
        assert lib.llmgpu_op_linear_fwd(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), 0, None, 0,
                                        0.0, None, 0, None, 0, None, 0, out.data_ptr(), 1, N, M, N, K,
                                        work, None, st) == 0
    assert torch.equal(y, ops.linear_fwd(x, w, out_dtype=F32)[0])
    assert bool((buf[n:] == 0xA5).all())
    xd, wd = x.double(), w.double().t()
    want, tol = xd @ wd, (K + 4) * ACC * (xd.abs() @ wd.abs())
    _close(y, want, tol, "with a workspace")
    _close(z, want, tol, "without")


_CAPTURED_FIRST = """
import torch
from llmgpu import ops
from llmgpu.ops import KernelError
dev = torch.device("cuda:0")
x = torch.ones(64, 64, dtype=torch.bfloat16, device=dev)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y, _ = ops.linear_fwd(x, x)
    word = ops._err_word(dev)
assert word, "the captured call has no error word"
g.replay()
ops.check_device(dev)
assert bool((y == 64).all()) and ops._err_word(dev) == word

class At:  # the word as a tensor
    __cuda_array_interface__ = dict(shape=(1,), typestr="<i4", data=(word, False), version=3)
w = torch.as_tensor(At(), device=dev)
assert int(w) == 0
w.fill_(7)
try:
    ops.check_device(dev)
except KernelError as e:
    assert "7" in str(e)
else:
    raise AssertionError("not raised")
assert int(w) == 0
ops.check_device(dev)
print("captured first: ok")
"""


def test_first_call_may_be_captured(cuda):
    """The first call of a process has its device's error word inside a capture too."""
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "llm-cpp_b200", "python"))
    r = subprocess.run([sys.executable, "-c", _CAPTURED_FIRST], env=env, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "captured first: ok" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("w_mn", [False, True])
def test_few_rows_offsets_past_32_bits(cuda, w_mn):
    """Weights of more than 2^31 elements under 3 rows: columns (and rows of dw) on both sides of it."""
    from llmgpu import ops
    M, K, N = 3, 32768, 70000
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(M, K, generator=g, device=cuda).to(BF)
    w = torch.empty((K, N) if w_mn else (N, K), dtype=BF, device=cuda)
    w.normal_(0, 0.01, generator=g)
    at = torch.tensor([0, 1, 40000, 65535, 65536, 65537, N - 1], device=cuda)  # of N
    wa = (w[:, at].t() if w_mn else w[at]).double()
    y, _ = ops.linear_fwd(x, w, w_mn=w_mn, out_dtype=F32)
    xd = x.double()
    _close(y[:, at], xd @ wa.t(), (K + 4) * ACC * (xd.abs() @ wa.abs().t()), "y")
    dy = torch.zeros(M, N, device=cuda)
    dy[:, at] = torch.randn(M, len(at), generator=g, device=cuda)
    dx, dw, _ = ops.linear_bwd(dy, x, w, w_mn=w_mn, dx_dtype=F32)
    dz = dy[:, at].double()
    _close(dx, dz @ wa, (H16 + (N + 4) * ACC) * (dz.abs() @ wa.abs()), "dx")
    want = dz.t() @ xd
    got = dw[:, at].t() if w_mn else dw[at]
    _close(got, want, H16 * want.abs() + (M + 4) * ACC * (dz.abs().t() @ xd.abs()), "dw")
    assert int(torch.count_nonzero(dw)) == int(torch.count_nonzero(got))
    ops.check_device(cuda)


def test_few_rows_far_apart(cuda):
    """Two rows whose distance passes 2^31 elements, in every matrix that has them."""
    from llmgpu import ops
    M, K, N, ld = 2, 264, 136, 2 ** 31 + 64
    buf = torch.zeros(M, ld, dtype=BF, device=cuda)
    g = torch.Generator().manual_seed(4)
    near = [_mat(g, M, n, BF, cuda)[0] for n in (K, N, N, N)]  # x, resid, dy, pre
    cut = [0, 512, 1024, 1536, 2048]
    far = [buf[:, c:c + m.shape[1]] for c, m in zip(cut, near)]
    for f, m in zip(far, near):
        f.copy_(m)
    out = buf[:, 2048:2048 + N]
    w, rng = _mat(g, N, K, BF, cuda, 0.1)[0], _rng(cuda)
    ops.linear_fwd(far[0], w, None, "silu", 0.3, rng, 1, far[1], out=out)
    assert torch.equal(out, ops.linear_fwd(near[0], w, None, "silu", 0.3, rng, 1, near[1])[0])
    got = ops.linear_bwd(far[2], far[0], w, far[3], "silu", 0.3, rng, 1)
    want = ops.linear_bwd(near[2], near[0], w, near[3], "silu", 0.3, rng, 1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for f, m in zip(far, near):
        assert torch.equal(f, m)
    ops.check_device(cuda)


def test_two_threads_at_once(cuda):
    """Calls from two threads, each on a stream of its own, give what one thread's give."""
    import threading
    from llmgpu import ops
    s = [_block_state(cuda, 10 + i, rows=300 + 40 * i, C=128, F=512, V=3000) for i in range(2)]
    rng = _rng(cuda, 1, 1)
    want = [_block(ops, q, rng) for q in s]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i].append(_block(ops, s[i], rng))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - shown by the assertion below
            failed.append(repr(e))
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for i in range(2):
        assert len(got[i]) == 10
        for r in got[i]:
            assert all(torch.equal(r[k], want[i][k]) for k in want[i])
    ops.check_device(cuda)


# ------------------------------------------------------------------------------------ refusals
def test_wrapper_refusals(cuda):
    from llmgpu import ops
    x, w = torch.zeros(6, 16, dtype=BF, device=cuda), torch.zeros(24, 16, dtype=BF, device=cuda)
    rng = _rng(cuda)
    t = torch.zeros(6, dtype=torch.int32, device=cuda)
    odd = torch.zeros(6, 17, dtype=BF, device=cuda)
    bad = [lambda: ops.dropout_fwd(x, 1.5, rng), lambda: ops.dropout_fwd(x, 0.5, None),
           lambda: ops.dropout_fwd(x, 0.5, rng.to(torch.int32)),
           lambda: ops.dropout_fwd(x.half(), 0.5, rng), lambda: ops.dropout_fwd(x.t(), 0.5, rng),
           lambda: ops.dropout_fwd(x, 0.5, rng, resid=w),
           lambda: ops.dropout_fwd(x, 0.5, rng, resid=x.float()),
           lambda: ops.dropout_fwd(x[0], 0.5, rng),
           lambda: ops.dropout_fwd(x, 0.5, rng, out=x.new_zeros(1, 16).expand(6, 16)),
           lambda: ops.linear_fwd(x, w, act="tanh"), lambda: ops.linear_fwd(x.float(), w),
           lambda: ops.linear_fwd(x, w, w_mn=True), lambda: ops.linear_fwd(odd[:, 1:], w),
           lambda: ops.linear_fwd(odd[:, :16], w), lambda: ops.linear_fwd(x, w, p=0.5),
           lambda: ops.linear_fwd(x, w, bias=torch.zeros(16, device=cuda)),
           lambda: ops.linear_fwd(x, w, resid=torch.zeros(6, 24, device=cuda)),
           lambda: ops.linear_fwd(x, w, out=torch.zeros(6, 23, dtype=BF, device=cuda)),
           lambda: ops.linear_bwd(torch.zeros(6, 24, device=cuda), x, w, act="gelu"),
           lambda: ops.linear_bwd(torch.zeros(6, 23, device=cuda), x, w),
           lambda: ops.linear_bwd(torch.zeros(6, 24, device=cuda), x, w, accumulate=True),
           lambda: ops.linear_bwd(torch.zeros(6, 24, device=cuda), x, w, accumulate=True,
                                  dw=torch.zeros_like(w), dbias=torch.zeros(24, device=cuda)),
           lambda: ops.linear_cross_entropy_fwd(x, w, t.long()),
           lambda: ops.linear_cross_entropy_fwd(x, w, t, 1.0),
           lambda: ops.linear_cross_entropy_fwd(x, w, t[:5]),
           lambda: ops.linear_cross_entropy_bwd(x, w, t, torch.zeros(6, device=cuda), piece=100),
           lambda: ops.linear_cross_entropy_bwd(x, w, t, torch.zeros(5, device=cuda)),
           lambda: ops.linear_cross_entropy_bwd(x, w, t, torch.zeros(6, device=cuda),
                                                dw=torch.zeros_like(w), accumulate=True)]
    for i, f in enumerate(bad):
        with pytest.raises(ops.KernelError):
            f()
            pytest.fail(f"call {i} was not refused")
