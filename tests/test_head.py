"""The learned head's operators (hwer/head.py) against plain implementations in 64 bits on the CPU.

Tolerances.  u(T) is half a step of type T (float32 2^-24, float16 2^-11, bfloat16 2^-8).  A value that is rounded once to T may be off by u(T)
relative; a float32 sum of n terms by about sqrt(n) u(float32) relative to the sum of the terms' magnitudes (roundings are independent), taken
eight times.  Where a rounded value enters a later sum, the sum of magnitudes times its u is added."""
import math

import numpy as np
import pytest
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U32 = U[torch.float32]
TINY = {torch.float32: 1e-37, torch.float16: 2.0 ** -24, torch.bfloat16: 1e-37}       # below the smallest normal value steps stay the same size
TYPES = [torch.float32, torch.float16, torch.bfloat16]
gpu = pytest.mark.gpu


def close(got, want, tol, what=""):
    got, want, tol = got.detach().double().cpu(), want.double(), torch.as_tensor(tol, dtype=torch.float64).expand(want.shape)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = int((bad.double() * ((got - want).abs() / tol.clamp_min(1e-300)).nan_to_num(1e9)).argmax())
        raise AssertionError("%s: %d of %d outside; worst at %d: got %r, want %r, tolerance %r" % (
            what, int(bad.sum()), bad.numel(), i, float(got.reshape(-1)[i]), float(want.reshape(-1)[i]), float(tol.reshape(-1)[i])))


def rnd(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape))


@pytest.fixture(scope="module")
def hw():
    import hwer
    from hwer import native
    native.lib()
    return hwer


# ---------------------------------------------------------------------------------------------------------------- the C entries' refusals (no GPU)
def test_c_entries_refuse_before_any_launch():
    import ctypes
    from hwer import native
    lib = native.lib()
    p = ctypes.c_void_p(4096)      # never read: every call below is refused
    big = 1 << 40
    E, W = native.HWER_EINVAL, native.HWER_EWORKSPACE
    norm = lambda **k: lib.hwer_rms_norm(*[{**dict(x=p, ldx=8, r=None, ldr=0, w=None, wt=0, n=2, d=8, t=0, eps=1e-6, y=p, ldy=8, h=None, ldh=0, st=None), **k}[n] for n in  # noqa: E731
                                           ("x", "ldx", "r", "ldr", "w", "wt", "n", "d", "t", "eps", "y", "ldy", "h", "ldh", "st")])
    for bad in (dict(x=None), dict(ldx=7), dict(t=3), dict(d=0), dict(n=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(y=None), dict(ldy=7), dict(w=p, wt=2),
                dict(r=p, ldr=8), dict(r=p, ldr=7, h=p, ldh=8)):
        assert norm(**bad) == E, bad
    assert norm(n=0, x=None) == 0
    assert lib.hwer_rms_norm_q8(p, 8, None, 0, None, 0, 2, 8, 0, 1, 1e-6, None, 8, p, None, 0, None) == E
    assert lib.hwer_rms_norm_q8(p, 8, None, 0, None, 0, 2, 8, 0, 1, 1e-6, p, 8, None, None, 0, None) == E
    back = lambda dw=p, w=p, ws=p, nb=big, **k: lib.hwer_rms_norm_backward(p, 8, p, 8, w, 0, None, 0, 2, 8, k.get("t", 0), 1e-6, k.get("dx", p), 8, dw, ws, nb, None)  # noqa: E731
    assert back(w=None) == E and back(dx=None) == E and back(t=9) == E and back(ws=None) == W and back(nb=8) == W
    mm = lambda a=p, lda=8, m=2, n=2, k=8, ldo=2, t=0, sa=p: lib.hwer_matmul_q8(a, lda, sa, p, 8, p, None, m, n, k, p, ldo, t, None)  # noqa: E731
    assert mm(a=None) == E and mm(lda=7) == E and mm(m=-1) == E and mm(k=131072, lda=131072) == E and mm(ldo=1) == E and mm(t=5) == E and mm(sa=None) == E
    assert mm(m=1 << 31) == E and mm(m=1 << 30, n=1 << 30, ldo=1 << 30) == E
    assert mm(m=0) == 0 and mm(n=0) == 0
    ce = lambda q=p, ldq=8, e=p, t=p, n=2, v=3, d=8, dt=0, scale=1.0, red=1, loss=p, ws=p, nb=big: lib.hwer_catalogue_ce(  # noqa: E731
        q, ldq, e, 8, None, t, n, v, d, dt, scale, red, p, p, loss, p, None, ws, nb, None)
    for bad in (dict(q=None), dict(ldq=7), dict(e=None), dict(t=None), dict(n=-1), dict(v=0), dict(d=0), dict(d=257, ldq=300), dict(dt=4), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("inf")), dict(scale=float("nan")), dict(red=3), dict(loss=None), dict(n=1 << 31), dict(v=1 << 31)):
        assert ce(**bad) == E, bad
    assert ce(ws=None) == W and ce(nb=16) == W
    cb = lambda grad=p, red=1, mean=p, dq=p, de=p, ldde=8, bias=None, db=None, nb=big: lib.hwer_catalogue_ce_backward(  # noqa: E731
        p, 8, p, 8, bias, p, 2, 3, 8, 0, 1.0, red, grad, p, p, mean, dq, 8, de, ldde, db, p, nb, None)
    assert cb(red=0, grad=None) == E and cb(mean=None) == E and cb(ldde=7) == E and cb(db=p) == E and cb(bias=p, db=p, de=None) == E and cb(red=7) == E and cb(nb=64) == W
    cg = lambda red=1, loss=p, dq=p, de=p, ldde=8, bias=None, db=None, ws=p: lib.hwer_catalogue_ce_grads(p, 8, p, 8, bias, p, 2, 3, 8, 0, 1.0, red, loss, dq, 8, de, ldde, db, ws, big, None)  # noqa: E731,E501
    assert cg(red=0) == E and cg(loss=None) == E and cg(dq=None) == E and cg(de=None) == E and cg(ldde=7) == E and cg(db=p) == E and cg(ws=None) == W
    assert lib.hwer_catalogue_ce_workspace_bytes(1, 1, 300, 0, 0, 0, 1) == 0 and lib.hwer_catalogue_ce_workspace_bytes(0, 1, 8, 0, 0, 0, 1) > 0


def test_python_entries_refuse_host_tensors_and_wrong_shapes(hw):
    from hwer import native
    x, q = torch.zeros(3, 8), torch.zeros(3, 8, dtype=torch.int8)
    with pytest.raises(native.HwerNativeError):
        hw.rms_norm(x)
    with pytest.raises(TypeError):
        hw.rms_norm(x.double())
    with pytest.raises(TypeError):
        hw.rms_norm([1.0])
    with pytest.raises(ValueError):
        hw.rms_norm(torch.zeros(3, 0))
    with pytest.raises(TypeError):
        hw.matmul_q8(x, x[:, 0], q, x[:, 0])
    with pytest.raises(native.HwerNativeError):
        hw.matmul_q8(q, x[:, 0], q, x[:, 0])
    with pytest.raises(native.HwerNativeError):
        hw.catalogue_cross_entropy(x, x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        hw.catalogue_cross_entropy(x, torch.zeros(4, 9), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        hw.catalogue_cross_entropy_grads(x, x, torch.zeros(3, dtype=torch.int64), reduction="none")


@gpu
def test_python_entries_refuse_on_the_device(hw):
    x, q, s = torch.zeros(3, 8, device="cuda"), torch.zeros(3, 8, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    for f, err in ((lambda: hw.rms_norm(x, eps=-1), ValueError), (lambda: hw.rms_norm(x, weight=s), ValueError), (lambda: hw.rms_norm(x, weight=torch.ones(8, device="cuda").half()), TypeError),
                   (lambda: hw.rms_norm(x, residual=x.half()), ValueError), (lambda: hw.rms_norm(x, residual=x[:2]), ValueError), (lambda: hw.rms_norm(x, residual=x.cpu()), ValueError),
                   (lambda: hw.rms_norm_grads(x.half(), x), ValueError), (lambda: hw.matmul_q8(q, s, q[:, :7], s), ValueError), (lambda: hw.matmul_q8(q, s[:2], q, s), ValueError),
                   (lambda: hw.matmul_q8(q, s, q, s.double()), ValueError), (lambda: hw.matmul_q8(q, s, q, s, out_dtype=torch.float64), TypeError),
                   (lambda: hw.catalogue_cross_entropy(x, x, t, scale=0), ValueError), (lambda: hw.catalogue_cross_entropy(x, x, t[:2]), ValueError),
                   (lambda: hw.catalogue_cross_entropy(x, x, t.float()), ValueError), (lambda: hw.catalogue_cross_entropy(x, x, t, bias=s[:2]), ValueError),
                   (lambda: hw.catalogue_cross_entropy(x, x, t, bias=s.double()), ValueError), (lambda: hw.catalogue_cross_entropy(x, x, t, reduction="max"), ValueError),
                   (lambda: hw.catalogue_cross_entropy(x, x[:0], t), ValueError), (lambda: hw.catalogue_cross_entropy(x, x.half(), t), ValueError),
                   (lambda: hw.catalogue_cross_entropy(torch.zeros(3, 257, device="cuda"), torch.zeros(3, 257, device="cuda"), t), ValueError),
                   (lambda: hw.catalogue_cross_entropy(x, x, t.cpu()), ValueError)):
        with pytest.raises(err):
            f()


# ---------------------------------------------------------------------------------------------------------------- norm
def norm_reference(h, w, eps):
    f = h.double()
    r = 1 / torch.sqrt((f * f).mean(-1, keepdim=True) + eps)
    return f * r * (1.0 if w is None else w.double()), r


# every way a row is held: 16 / 64 / 256 / 1024 lanes, whole vectors and single elements, and rows too wide for registers
NORM_SHAPES = [(1, 1), (3, 2), (5, 7), (33, 16), (7, 64), (130, 100), (64, 250), (9, 256), (2, 511), (65, 512), (3, 1000), (5, 1024), (3, 1028), (4, 2048), (2, 2050), (3, 4096),
               (2, 4100), (3, 8192), (2, 12288), (2, 16384), (2, 16392), (2, 20001), (2, 40960), (5000, 24)]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d", NORM_SHAPES)
def test_norm_forward_and_gradients(hw, n, d, dtype):
    for wtype, with_res, with_dh in ((dtype, True, True), (torch.float32, False, False), (None, True, False)):
        x, res, dy, dh = (rnd(10 * n + d + i, n, d).to(dtype) for i in range(4))
        w = None if wtype is None else (1 + 0.3 * rnd(5, d)).to(wtype)
        eps = 1e-5
        xg, rg, wg = x.cuda(), res.cuda() if with_res else None, None if w is None else w.cuda()
        out = hw.rms_norm(xg, wg, rg, eps=eps)
        y, h = out if with_res else (out, xg)
        if with_res:      # one rounding of an exact-to-float32 sum
            assert torch.equal(h.cpu(), (x.float() + res.float()).to(dtype))
        hc = h.cpu()
        want, r = norm_reference(hc, w, eps)
        sums = 8 * math.sqrt(d) * U32
        close(y, want, want.abs() * (U[dtype] + sums + 6 * U32) + TINY[dtype], "y")
        dx, dw = hw.rms_norm_grads(dy.cuda(), h, wg, eps=eps, dh=dh.cuda() if with_dh else None)
        g = dy.double() * (1.0 if w is None else w.double())
        f = hc.double()
        back = (g * f).mean(-1, keepdim=True)
        want = r * (g - f * r * r * back) + (dh.double() if with_dh else 0)
        size = r * (g.abs() + f.abs() * r * r * (g * f).abs().mean(-1, keepdim=True)) + (dh.double().abs() if with_dh else 0)
        close(dx, want, want.abs() * U[dtype] + size * (2 * sums + 8 * U32) + TINY[dtype], "dx")
        if w is None:
            assert dw is None
        else:
            terms = dy.double() * f * r
            close(dw, terms.sum(0), terms.sum(0).abs() * U[w.dtype] + terms.abs().sum(0) * (8 * math.sqrt(n) * U32 + sums + 8 * U32) + TINY[w.dtype], "dweight")


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d", [(20011, 40), (7001, 1030), (2900, 4104), (1100, 20000), (40000, 3)])
def test_norm_of_many_rows(hw, n, d, dtype):
    """the weights' gradient joined from many workgroups' parts"""
    test_norm_forward_and_gradients(hw, n, d, dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_norm_gradients_against_differences(hw, dtype):
    """The gradient of sum(y * c) + sum(h * k) along a direction against the difference of the 64-bit formula on both sides."""
    x, res, c, k, v = (rnd(70 + i, 6, 40) for i in range(5))
    w = 1 + 0.2 * rnd(80, 40)
    x, res, c, k, w = (t.to(dtype) for t in (x, res, c, k, w))
    h = (x.float() + res.float()).to(dtype).double()
    xg, rg, wg = (t.cuda().requires_grad_() for t in (x, res, w))
    y, hh = hw.rms_norm(xg, wg, rg, eps=1e-4)
    torch.autograd.backward([y, hh], [c.cuda(), k.cuda()])
    assert torch.equal(xg.grad, rg.grad)
    f = lambda a, b: (norm_reference(a, b, 1e-4)[0] * c.double()).sum() + (a * k.double()).sum()  # noqa: E731
    t = 1e-5
    want = (f(h + t * v, w.double()) - f(h - t * v, w.double())) / (2 * t)
    got = (xg.grad.cpu().double() * v).sum()
    # each of the 240 gradients is rounded once
    assert abs(got - want) <= 2 * U[dtype] * (xg.grad.cpu().double() * v).abs().sum() + 1e-6
    z = rnd(81, 40)
    want = (f(h, w.double() + t * z) - f(h, w.double() - t * z)) / (2 * t)
    got = (wg.grad.cpu().double() * z).sum()
    assert abs(got - want) <= 2 * U[dtype] * (wg.grad.cpu().double() * z).abs().sum() + 1e-6


@gpu
def test_norm_autograd_uses(hw):
    """which inputs require a gradient, which outputs are used, leading dimensions, strided and broadcast inputs"""
    x = rnd(1, 2, 3, 32).float()
    w = (1 + 0.1 * rnd(2, 32)).float()
    for need in ((True, True), (True, False), (False, True)):
        xg, wg = x.cuda().requires_grad_(need[0]), w.cuda().requires_grad_(need[1])
        y = hw.rms_norm(xg, wg)
        assert y.shape == x.shape
        y.square().sum().backward()
        xc, wc = x.double().requires_grad_(need[0]), w.double().requires_grad_(need[1])
        norm_reference(xc, wc, 1e-6)[0].square().sum().backward()
        for a, b in ((xg, xc), (wg, wc)):
            assert (a.grad is None) == (b.grad is None)
            if a.grad is not None:
                close(a.grad, b.grad, 1e-4 * (1 + b.grad.abs()))
    xg, wg, rg = x.cuda().requires_grad_(), w.cuda().requires_grad_(), x.cuda().requires_grad_()
    hw.rms_norm(xg, wg, rg)[1].sum().backward()          # only the sum is used
    assert torch.equal(xg.grad.cpu(), torch.ones_like(x)) and torch.equal(rg.grad, xg.grad) and float(wg.grad.abs().max()) == 0
    wide = rnd(3, 6, 96).float().cuda()
    view = wide[:, 32:64]                                  # rows of a wider table: not on 16 bytes behind each other, read in place
    assert torch.equal(hw.rms_norm(view), hw.rms_norm(view.contiguous()))
    shifted = rnd(4, 6 * 40 + 1).float().cuda()[1:].reshape(6, 40)      # not on 16 bytes
    assert torch.allclose(hw.rms_norm(shifted), hw.rms_norm(shifted.clone()), rtol=1e-6)
    assert torch.equal(hw.rms_norm(wide.t()), hw.rms_norm(wide.t().contiguous()))
    row = wide[:1].expand(6, 96)
    assert torch.equal(hw.rms_norm(row), hw.rms_norm(row.contiguous()))
    one = wide[:1].clone().requires_grad_()
    hw.rms_norm(one.expand(6, 96)).sum().backward()        # a broadcast input: the gradients of its copies are added
    six = wide[:1].clone().requires_grad_()
    (6 * hw.rms_norm(six)).sum().backward()
    assert torch.allclose(one.grad, six.grad, rtol=1e-4, atol=1e-5)
    e = torch.zeros(0, 32, device="cuda").requires_grad_()
    y = hw.rms_norm(e, wg)
    wg.grad = None
    y.sum().backward()
    assert y.shape == (0, 32) and float(wg.grad.abs().max()) == 0


def codes_reference(h, w):
    v = h.double() * (1.0 if w is None else w.double())
    top = v.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * v / top), 0).to(torch.int8), top[..., 0]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d", NORM_SHAPES)
def test_q8_codes_are_exact(hw, n, d, dtype):
    for wtype, with_res in ((dtype, True), (torch.float32, False), (None, False)):
        x, res = rnd(n + 3 * d, n, d).to(dtype), rnd(n + 3 * d + 1, n, d).to(dtype)
        if d > 8:
            # borders between two codes: with the row's largest value 127 * 2^-k, (c + 1/2) * 2^-k is exactly between c and c + 1
            x[0, 0] = 127 / 16
            x[0, 1:9] = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, 3.5, 100.5, -126.5]) / 16
            x[0, 9:] = x[0, 9:].clamp(-1, 1)
            if with_res:
                res[0] = 0
        w = None if wtype is None else (1 + 0.3 * rnd(5, d)).to(wtype)
        if w is not None and d > 8:
            w[:9] = 1
            w[9:] = w[9:].clamp(-2, 2)
        wg = None if w is None else w.cuda()
        out = hw.rms_norm_q8(x.cuda(), wg, res.cuda() if with_res else None, eps=1e-5)
        h = x if not with_res else (x.float() + res.float()).to(dtype)
        if with_res:
            assert torch.equal(out[2].cpu(), h)
        codes, top = codes_reference(h, w)
        assert torch.equal(out[0].cpu(), codes)
        _, r = norm_reference(h, w, 1e-5)
        want = top * r[:, 0] / 127
        close(out[1], want, want * (8 * math.sqrt(d) * U32 + 8 * U32), "scale")
        q, s = hw.quantize_rows_q8(x.cuda())
        codes, top = codes_reference(x, None)
        assert torch.equal(q.cpu(), codes)
        close(s, top / 127, top / 127 * 3 * U32, "scale of plain codes")


@gpu
@pytest.mark.parametrize("d", [24, 4096, 40961])
def test_q8_and_norm_special_rows(hw, d):
    x = rnd(1, 6, d).float()
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    x[3] *= 1e-42                       # denormal values
    x[4, 0], x[4, 1:] = 1e30, 1e-30     # everything else far below half a step
    x[3, 0] = 3e-42
    q, s = hw.quantize_rows_q8(x.cuda())
    q, s = q.cpu(), s.cpu()
    assert (q[:3] == 0).all() and s[0] == 0 and torch.isnan(s[1]) and torch.isnan(s[2])
    codes, top = codes_reference(x, None)
    assert torch.equal(q[3:], codes[3:])
    assert abs(float(s[4]) - 1e30 / 127) <= 1e30 / 127 * 3 * U32
    y = hw.rms_norm(x.cuda(), eps=0.0).cpu()
    assert torch.isnan(y[0]).all() and torch.isnan(y[1]).all() and torch.isnan(y[2, 5]) and torch.isfinite(y[5]).all()
    y = hw.rms_norm(x.cuda(), eps=1e-6).cpu()
    assert (y[0] == 0).all() and torch.isfinite(y[3]).all()


# ---------------------------------------------------------------------------------------------------------------- 8-bit product
def q8(seed, n, k):
    return torch.from_numpy(np.random.default_rng(seed).integers(-128, 128, (n, k), dtype=np.int8))


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 5, 3), (1, 300, 64), (2, 1000, 250), (16, 33, 128), (17, 70, 144), (33, 65, 1000), (64, 4096, 512), (65, 65, 16), (65, 129, 0), (1, 4, 0),
                                    (300, 1, 77), (1000, 40, 256), (128, 128, 128), (129, 257, 100), (200, 1682, 64), (943, 1682, 64), (257, 511, 1040), (130, 130, 4096), (100, 90, 131071)])
def test_matmul_q8(hw, m, n, k):
    a, b = q8(m + k, m, k), q8(n + k + 1, n, k)
    sa, sb, bias = (rnd(i, r).float().abs() + 0.01 for i, r in ((1, m), (2, n), (3, n)))
    ints = (a.double() @ b.double().t())      # exact: below 2^31
    for dtype, with_bias in ((torch.float32, True), (torch.bfloat16, False), (torch.float16, True)):
        s = 2.0 ** -12 if dtype == torch.float16 else 1.0      # inside float16's range
        out = hw.matmul_q8(a.cuda(), (sa * s).cuda(), b.cuda(), (sb * s).cuda(), (bias * s * s).cuda() if with_bias else None, out_dtype=dtype)
        size = (ints * sa[:, None].double() * sb.double()) * s * s
        want = size + (bias.double() * s * s if with_bias else 0)
        # the integer's rounding to float32, two products, a sum; then the output's type
        close(out, want, want.abs() * (U[dtype] + U32) + size.abs() * 3 * U32 + TINY[dtype], str(dtype))


@gpu
@pytest.mark.parametrize("k", [64, 250, 257, 272, 384, 512, 640, 1000, 1280])
@pytest.mark.parametrize("m,n,views", [(33, 70, "whole"), (32, 70, "whole"), (70, 31, "whole"), (100, 450, "whole"), (1600, 2000, "whole"), (2900, 4200, "whole"),
                                       (100, 450, "odd"), (1600, 2001, "odd"), (2900, 4200, "odd"), (24, 450, "odd"), (3003, 6001, "whole"), (3003, 6001, "odd")])
def test_matmul_q8_tiles(hw, m, n, k, views):
    """every size of tile, with fewer steps of K than it has buffers and more, partial last steps, partial tiles; rows on 16 bytes and not"""
    from hwer import native
    a, b = q8(m + k, m, k).cuda(), q8(n + k + 1, n, k).cuda()
    if views == "odd":
        a, b = (torch.cat([t.new_full((t.shape[0], 1), 77), t, t.new_full((t.shape[0], 2), -99)], 1)[:, 1:-2] for t in (a, b))
    sa, sb = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    buf = torch.full((m + 1, n + 5), 7.0, device="cuda")
    out = buf[:m, 2:2 + n]
    lib = native.lib()
    assert lib.hwer_matmul_q8(a.data_ptr(), a.stride(0), sa.data_ptr(), b.data_ptr(), b.stride(0), sb.data_ptr(), None, m, n, k, out.data_ptr(), n + 5, 0, torch.cuda.current_stream().cuda_stream) == 0
    want = a.double() @ b.double().t()      # below 2^24 in magnitude at these K with scales of one: exact in float32
    assert want.abs().max() < 2 ** 24 and torch.equal(out.double(), want)
    assert (buf[m] == 7).all() and (buf[:, :2] == 7).all() and (buf[:, 2 + n:] == 7).all()
    got = hw.matmul_q8(a, sa, b, sb, out_dtype=torch.bfloat16)
    assert torch.equal(got, want.float().bfloat16())


@gpu
def test_matmul_q8_strides_and_order(hw):
    """rows of a wider table, rows that are not on 16 bytes, a transposed operand; the same product with the sides exchanged is the same, bit for bit"""
    a, b = q8(1, 100, 300).cuda(), q8(2, 200, 300).cuda()
    sa, sb = torch.rand(100, device="cuda") + 0.1, torch.rand(200, device="cuda") + 0.1
    want = hw.matmul_q8(a[:, 16:272].contiguous(), sa, b[:, 16:272].contiguous(), sb)
    assert torch.equal(want, hw.matmul_q8(a[:, 16:272], sa, b[:, 16:272], sb))
    at = a[:, 16:272].t().contiguous().t()
    assert torch.equal(want, hw.matmul_q8(at, sa, b[:, 16:272], sb))
    odd = torch.empty(100 * 256 + 3, dtype=torch.int8, device="cuda")[3:].view(100, 256).copy_(a[:, 16:272])
    assert torch.equal(want, hw.matmul_q8(odd, sa, b[:, 16:272], sb))
    few = hw.matmul_q8(a[:10, 16:272].contiguous(), sa[:10], b[:, 16:272].contiguous(), sb)
    assert torch.equal(few, want[:10])                     # the short-side kernel and the tiles
    ones = torch.ones_like(sa)
    swapped = hw.matmul_q8(b[:, 16:272], torch.ones_like(sb), a[:10, 16:272], ones[:10])
    assert torch.equal(swapped.t(), hw.matmul_q8(a[:10, 16:272], ones[:10], b[:, 16:272], torch.ones_like(sb)))
    bad = sb.clone()
    bad[7] = float("nan")
    out = hw.matmul_q8(a[:, 16:272], sa, b[:, 16:272], bad)
    assert torch.isnan(out[:, 7]).all() and torch.equal(out[:, 8:], want[:, 8:])


# ---------------------------------------------------------------------------------------------------------------- cross entropy
def ce_reference(x, e, t, s, bias, g):
    """(rows' losses, lse, dx, de, db, and the sums of magnitudes behind each gradient) for gradients g of the rows' losses"""
    x, e = x.double(), e.double()
    z = s * (x @ e.t())
    if bias is not None:
        z = z + bias.double()
    top = z.amax(1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    ex = torch.exp(z - top)
    total = ex.sum(1, keepdim=True)
    lse = torch.log(total)[:, 0] + top[:, 0]
    p = torch.where(total > 0, ex / total, torch.zeros_like(ex))
    on = (t >= 0) & (t < len(e))
    at = t.clamp(0, len(e) - 1)
    rows = torch.where(on, lse - z.gather(1, at[:, None])[:, 0], torch.where(t == -1, 0.0, float("nan")))
    rows = torch.where(on & (total[:, 0] == 0), torch.full_like(rows, float("inf")), rows)
    gw = torch.where(on, g, torch.zeros_like(g))[:, None]
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    w, wa = gw * (p - hot), gw.abs() * (p + hot)
    wd = gw.abs() * p      # the part that is rounded to the rows' type
    return dict(rows=rows, lse=lse, dx=s * (w @ e), de=s * (w.t() @ x), db=w.sum(0), dx_size=s * (wa @ e.abs()), de_size=s * (wa.t() @ x.abs()), db_size=wa.sum(0),
                dx_low=s * gw.abs() * p.amax(1, keepdim=True) * e.abs().sum(0), de_low=s * (gw.abs().t() @ x.abs()), dx_p=s * (wd @ e.abs()), de_p=s * (wa.t() @ x.abs()), z_size=s * (x.abs() @ e.abs().t()).amax(1) + (0 if bias is None else bias.double().abs().nan_to_num(0, 0, 0).clamp_max(1e3).amax()))


def ce_tolerances(ref, dtype, n, v, d, rows_loss=True):
    u = U[dtype]
    # a logit: d products (float32 rows: three of two float16 terms, 3 * 2^-22 each) summed in float32; a probability: twice that and the sum's roundings
    dz = ref["z_size"].max().item() * ((9 * 2.0 ** -22 if dtype == torch.float32 else 0) + 8 * math.sqrt(3 * d) * U32 + 4 * U32)
    dp = 2 * dz + (8 * math.sqrt(v) + 32) * U32
    w = 2.0 ** -22 if dtype == torch.float32 else u          # the weights' rounding for the second product
    # ... in float16 (float32 rows: two terms of it), where small weights keep an absolute half step of 2^-25: after the factor that they carry 2^-36 of
    # the row's largest probability for the queries' gradient, 2^-40 of the largest gradient of a row for the table's
    low = (0.0, 0.0) if dtype == torch.bfloat16 else (2.0 ** -36, 2.0 ** -40)
    return dict(loss=2 * dz + (8 * math.sqrt(v) + 32) * U32,
                dx=ref["dx"].abs() * u + ref["dx_p"] * w + ref["dx_size"] * (dp + 8 * math.sqrt(3 * v) * U32) + ref["dx_low"] * low[0] + 4 * TINY[dtype],
                de=ref["de"].abs() * u + ref["de_p"] * w + ref["de_size"] * (dp + 8 * math.sqrt(3 * n) * U32) + ref["de_low"] * low[1] + 4 * TINY[dtype],
                db=ref["db_size"] * (dp + 8 * math.sqrt(n) * U32) + 1e-30)


def ce_inputs(seed, n, v, d, dtype, bias=False, spread=1.0):
    x, e = rnd(seed, n, d) / math.sqrt(d), rnd(seed + 1, v, d) / math.sqrt(d)
    e = e * torch.exp(spread * rnd(seed + 2, v, 1))
    t = torch.from_numpy(np.random.default_rng(seed + 3).integers(0, v, n))
    b = rnd(seed + 4, v).float() if bias else None
    return x.to(dtype), e.to(dtype), t, b


def ce_check(hw, x, e, t, s, b, reduction="mean"):
    n, d = x.shape
    v = len(e)
    counted = max(1, int((t != -1).sum()))
    g = torch.full((n,), 1.0 / counted if reduction == "mean" else 1.0, dtype=torch.float64)
    ref = ce_reference(x, e, t, s, b, g)
    tol = ce_tolerances(ref, x.dtype, n, v, d)
    dev = [None if a is None else a.cuda() for a in (x, e, t, b)]
    out = hw.catalogue_cross_entropy_grads(dev[0], dev[1], dev[2], scale=s, bias=dev[3], reduction=reduction)
    want = ref["rows"].sum() / (counted if reduction == "mean" else 1)
    close(out[0], want, tol["loss"] * (1 if reduction == "mean" else n) + want.abs() * 2 * U32, "loss")
    close(out[1], ref["dx"], tol["dx"], "dqueries")
    close(out[2], ref["de"], tol["de"], "dtable")
    if b is not None:
        close(out[3], ref["db"], tol["db"], "dbias")
    assert torch.equal(out[0], hw.catalogue_cross_entropy(dev[0], dev[1], dev[2], scale=s, bias=dev[3], reduction=reduction))
    rows = hw.catalogue_cross_entropy(dev[0], dev[1], dev[2], scale=s, bias=dev[3], reduction="none")
    close(rows, ref["rows"], tol["loss"] + ref["rows"].abs() * U32, "rows")
    return out


CE_SHAPES = [(1, 1, 1), (1, 2, 3), (1, 129, 64), (2, 33, 128), (33, 32, 64), (31, 65, 100), (129, 127, 128), (64, 500, 250), (130, 1000, 256), (200, 300, 17), (257, 1682, 64), (1, 5000, 96),
             (700, 3, 66), (1500, 70, 128), (300, 2048, 256)]


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", CE_SHAPES)
def test_cross_entropy_and_gradients(hw, n, v, d, dtype):
    x, e, t, b = ce_inputs(n + v + d, n, v, d, dtype)
    ce_check(hw, x, e, t, 6.0, None)
    t[::3] = -1
    ce_check(hw, x, e, t, 0.7, rnd(9, v).float(), reduction="sum")


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(1000, 30000, 64), (16, 150000, 96), (200, 40000, 250), (9000, 300, 128), (5000, 129, 256), (2500, 4000, 100), (70, 20000, 3)])
def test_cross_entropy_split_over_either_side(hw, n, v, d, dtype):
    """a few and hundreds of splits in both passes, and their joins; rows with gradients of their own, of which some are zero"""
    x, e, t, b = ce_inputs(n + v + d, n, v, d, dtype, bias=True)
    t[::5] = -1
    b[::11] = float("-inf")
    t = torch.where(t % 11 == 0, t + 1, t).clamp_max(v - 1 if (v - 1) % 11 else v - 2)
    up = rnd(7, n)
    up[::4] = 0
    up[1::8] *= 1e-4
    ref = {k: a.cpu() for k, a in ce_reference(x.cuda(), e.cuda(), t.cuda(), 4.0, b.cuda(), up.cuda()).items()}
    tol = ce_tolerances(ref, dtype, n, v, d)
    xs, es, bs = x.cuda().requires_grad_(), e.cuda().requires_grad_(), b.cuda().requires_grad_()
    rows = hw.catalogue_cross_entropy(xs, es, t.cuda(), scale=4.0, bias=bs, reduction="none")
    close(rows, ref["rows"], tol["loss"] + ref["rows"].abs() * U32, "rows")
    rows.backward(up.float().cuda())
    # a row's gradient enters in float32, relative to the largest: two more roundings; in float16 a weight of the table's sum keeps 2^-40 of the largest
    # gradient's (not of its own row's)
    floor = 0.0 if dtype == torch.bfloat16 else 2.0 ** -40 * 4.0 * up.abs().max() * x.double().abs().sum(0)
    close(xs.grad, ref["dx"], tol["dx"] + ref["dx_size"] * 4 * U32, "dqueries")
    close(es.grad, ref["de"], tol["de"] + ref["de_size"] * 4 * U32 + floor, "dtable")
    close(bs.grad, ref["db"], tol["db"] + ref["db_size"] * 4 * U32, "dbias")
    again = [a.detach().clone().requires_grad_() for a in (xs, es, bs)]
    hw.catalogue_cross_entropy(again[0], again[1], t.cuda(), scale=4.0, bias=again[2], reduction="none").backward(up.float().cuda())
    assert all(torch.equal(p.grad, q.grad) for p, q in zip(again, (xs, es, bs)))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_cross_entropy_sharp_and_flat_rows(hw, dtype):
    """logits that rise along the catalogue (the running maximum is renewed all the way), one class that takes everything, and equal logits"""
    n, v, d = 70, 700, 64
    x, e, t, _ = ce_inputs(3, n, v, d, dtype, spread=0)
    e[:, 0] = torch.linspace(-2, 6, v).to(dtype)
    x[:, 0] = torch.linspace(-3, 3, n).to(dtype)
    ce_check(hw, x, e, t, 8.0, None)
    ce_check(hw, x, e, t, 8.0, torch.linspace(5, -20, v))
    ce_check(hw, torch.zeros_like(x), e, t, 8.0, None)          # every row uniform
    ce_check(hw, x, e, torch.full_like(t, 5), 3.0, None)        # the same class again and again


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(64, 2, 64), (50, 9, 100), (70, 300, 128), (33, 1, 64)])
def test_cross_entropy_of_learnt_rows_keeps_its_digits(hw, n, v, d, dtype):
    """losses of 1e-2 .. 1e-8: everything is proportional to 1 - p_t, and accurate relative to it"""
    e = (rnd(1, v, d) / math.sqrt(d)).to(dtype)
    t = torch.arange(n) % v
    x = (e.double()[t] + 0.05 * rnd(2, n, d) / math.sqrt(d)).to(dtype)
    s = 16.0
    for b in (None, 0.1 * rnd(4, v).float()):
        g = torch.full((n,), 1.0 / n, dtype=torch.float64)
        ref = ce_reference(x, e, t, s, b, g)
        z = s * (x.double() @ e.double().t()) + (0 if b is None else b.double())
        others = torch.softmax(z, 1).scatter(1, t[:, None], 0.0)
        miss = others.sum(1)
        hot = torch.zeros_like(others).scatter(1, t[:, None], 1.0)
        rows = torch.log1p(torch.exp(torch.logsumexp(z.masked_fill(hot > 0, -math.inf), 1) - z.gather(1, t[:, None])[:, 0]))
        if v > 9:
            assert rows.median() < 2e-2
        dz = ce_tolerances(ref, dtype, n, v, d)["loss"]
        u, w = U[dtype], 2.0 ** -22 if dtype == torch.float32 else U[dtype]
        low = 0.0 if dtype == torch.bfloat16 else 2.0 ** -36
        mags = lambda o, m: s / n * (o @ e.double().abs() + m[:, None] * e.double().abs()[t])  # noqa: E731
        dx = s / n * (others @ e.double() - miss[:, None] * e.double()[t])
        wt = others + hot * miss[:, None]
        de = s / n * ((others - hot * miss[:, None]).t() @ x.double())
        de_size = s / n * (wt.t() @ x.double().abs())
        dev = [None if a is None else a.cuda() for a in (x, e, t, b)]
        out = hw.catalogue_cross_entropy_grads(dev[0], dev[1], dev[2], scale=s, bias=dev[3])
        got = hw.catalogue_cross_entropy(dev[0], dev[1], dev[2], scale=s, bias=dev[3], reduction="none")
        close(got, rows, rows * (4 * dz + 1e-6) + 1e-37, "rows")
        floor = s / n * low * (others.amax(1, keepdim=True) * e.double().abs().sum(0))
        close(out[1], dx, dx.abs() * u + mags(others, miss) * (w + 4 * dz + 1e-6) + floor + 4 * TINY[dtype], "dx")
        # (in float16 the weights' steps stay at 2^-24 below 2^-14: an absolute 2^-40 after the factor 2^15)
        close(out[2], de, de.abs() * u + de_size * (w + 4 * dz + 1e-6) + (s * 2.0 ** -40 * x.double().abs().mean(0) if low else 0) + 4 * TINY[dtype], "de")


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_cross_entropy_masks(hw, dtype):
    n, v, d = 40, 333, 96
    x, e, t, b = ce_inputs(21, n, v, d, dtype, bias=True)
    b[::7] = float("-inf")
    b[:64] = float("-inf")                    # whole tiles without a class
    t = torch.where(torch.isinf(b[t]), torch.tensor(65), t)
    assert not torch.isinf(b[65])
    out = ce_check(hw, x, e, t, 4.0, b)
    assert float(out[3].cpu()[torch.isinf(b)].abs().max()) == 0 and float(out[2].cpu().float()[torch.isinf(b)].abs().max()) == 0
    # a class whose offset is float32's lowest value is as good as gone, unless nothing else is left: then all are equal
    low = torch.full((v,), torch.finfo(torch.float32).min)
    part = torch.where(torch.arange(v) < 200, low, torch.zeros(v))
    ce_check(hw, x, e, t.clamp_min(200), 4.0, part)
    rows = hw.catalogue_cross_entropy(x.cuda(), e.cuda(), t.cuda(), scale=4.0, bias=low.cuda(), reduction="none")
    assert torch.equal(rows.cpu().isnan(), torch.zeros(n, dtype=torch.bool)) and float(rows.cpu().max()) < 1e32
    # nothing left at all
    loss, dx, de, db = hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), t.cuda(), scale=4.0, bias=torch.full((v,), float("-inf")).cuda())
    assert float(loss) == float("inf") and torch.isfinite(dx).all() and torch.isfinite(de).all() and torch.isfinite(db).all()
    # the target itself masked: an infinite loss, the formula's gradient
    t2 = t.clone()
    t2[0] = 0
    rows = hw.catalogue_cross_entropy(x.cuda(), e.cuda(), t2.cuda(), scale=4.0, bias=b.cuda(), reduction="none").cpu()
    assert rows[0] == float("inf") and torch.isfinite(rows[1:]).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(70, 333, 64), (300, 150, 128), (129, 1000, 100), (40, 500, 256)])
def test_cross_entropy_unused_rows_hold_anything(hw, n, v, d, dtype):
    """NaN, infinities and huge values in queries that do not count (padding) and in classes that are taken out: the same as zeros there, bit for bit"""
    x, e, t, b = ce_inputs(n + d, n, v, d, dtype, bias=True)
    b[3::7] = float("-inf")
    t = torch.where(torch.isinf(b[t]), t - 1, t)
    t[::3] = -1
    t[-1] = -1
    top = torch.finfo(dtype).max
    bad_x, bad_e, clean_x, clean_e = x.clone(), e.clone(), x.clone(), e.clone()
    clean_x[t == -1], clean_e[torch.isinf(b)] = 0, 0
    for i, value in enumerate((float("nan"), float("inf"), -float("inf"), top, -top)):
        bad_x[torch.nonzero(t == -1)[i::5, 0], i::3] = value
        bad_e[torch.nonzero(torch.isinf(b))[i::5, 0], i::4] = value
    t = t.cuda()
    for queries, table, bias in (((bad_x, clean_x), (e, e), None), ((bad_x, clean_x), (bad_e, clean_e), b.cuda())):
        got, want = ([], [])
        for out, q, tab in ((got, queries[0].cuda(), table[0].cuda()), (want, queries[1].cuda(), table[1].cuda())):
            out.extend(hw.catalogue_cross_entropy_grads(q, tab, t, scale=4.0, bias=bias))
            out.append(hw.catalogue_cross_entropy(q, tab, t, scale=4.0, bias=bias, reduction="none"))
            for reduction in ("mean", "none"):
                leaves = [None if a is None else a.clone().requires_grad_() for a in (q, tab, bias)]
                loss = hw.catalogue_cross_entropy(leaves[0], leaves[1], t, scale=4.0, bias=leaves[2], reduction=reduction)
                up = torch.linspace(-1, 1, n, device="cuda")
                if out is got:      # and so may the gradients that reach them
                    up[t == -1] = torch.tensor([float("inf"), float("nan"), 1e30], device="cuda").repeat(n)[:int((t == -1).sum())]
                loss.backward(up if reduction == "none" else None)
                out.extend([loss.detach()] + [a.grad for a in leaves if a is not None])
        assert all(torch.isfinite(a).all() and torch.equal(a, c) for a, c in zip(got, want))
        close(want[0], ce_reference(queries[1], table[1], t.cpu(), 4.0, None if bias is None else b, torch.ones(n, dtype=torch.float64))["rows"].sum() / int((t >= 0).sum()), 2e-3 if dtype != torch.float32 else 1e-4)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_cross_entropy_a_bad_row_stays_alone(hw, dtype):
    """a counted query with an infinity or NaN: its own loss and gradient are lost (and the sums it enters), the other rows' are not"""
    n, v, d = 50, 200, 64
    x, e, t, _ = ce_inputs(11, n, v, d, dtype)
    want = hw.catalogue_cross_entropy(x.cuda(), e.cuda(), t.cuda(), scale=4.0, reduction="none")
    y = x.clone()
    y[7, 3], y[20, 5] = float("inf"), float("nan")
    q = y.cuda().requires_grad_()
    got = hw.catalogue_cross_entropy(q, e.cuda(), t.cuda(), scale=4.0, reduction="none")
    keep = torch.ones(n, dtype=torch.bool)
    keep[[7, 20]] = False
    assert torch.equal(got.detach()[keep], want[keep]) and not torch.isfinite(got.detach()[~keep]).any()
    got[keep.cuda()].sum().backward()
    assert torch.isfinite(q.grad[keep]).all()


@gpu
def test_cross_entropy_targets(hw):
    """rows that do not count, no row that counts, no row at all, and targets that name nothing"""
    x, e, t, _ = ce_inputs(5, 50, 90, 64, torch.float32)
    t[10:20] = -1
    loss, dx, de = ce_check(hw, x, e, t, 2.0, None)
    assert float(dx[10:20].abs().max()) == 0
    loss, dx, de = hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), torch.full_like(t, -1).cuda())
    assert float(loss) == 0 and float(dx.abs().max()) == 0 and float(de.abs().max()) == 0
    for red, want in (("mean", 0.0), ("sum", 0.0)):
        loss, dx, de = hw.catalogue_cross_entropy_grads(x[:0].cuda(), e.cuda(), t[:0].cuda(), reduction=red)
        assert float(loss) == want and dx.shape == (0, 64) and float(de.abs().max()) == 0
    assert hw.catalogue_cross_entropy(x[:0].cuda(), e.cuda(), t[:0].cuda(), reduction="none").shape == (0,)
    t2 = t.clone()
    t2[3], t2[4], t2[5] = 90, -2, 1 << 40
    rows = hw.catalogue_cross_entropy(x.cuda(), e.cuda(), t2.cuda(), reduction="none").cpu()
    assert torch.isnan(rows[3:6]).all() and torch.isfinite(rows[:3]).all() and torch.isfinite(rows[6:]).all()
    loss, dx, de = hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), t2.cuda())
    assert math.isnan(float(loss)) and float(dx[3:6].abs().max()) == 0 and torch.isfinite(de).all()
    a = hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), t.cuda())
    b = hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), t.to(torch.int32).cuda())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_cross_entropy_strides(hw, dtype):
    """rows of a wider table and rows that are not on 16 bytes give the same as their copies"""
    x, e, t, _ = ce_inputs(31, 70, 200, 128, dtype)
    want = hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), t.cuda(), scale=3.0)
    wx, we = torch.randn(70, 160, device="cuda").to(dtype), torch.randn(200, 131, device="cuda").to(dtype)
    wx[:, 16:144], we[:, 3:131] = x.cuda(), e.cuda()
    for q, tab in ((wx[:, 16:144], e.cuda()), (x.cuda(), we[:, 3:131]), (wx[:, 16:144], we[:, 3:131]), (x.t().contiguous().cuda().t(), e.cuda())):
        got = hw.catalogue_cross_entropy_grads(q, tab, t.cuda(), scale=3.0)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_autograd(hw, dtype, reduction):
    n, v, d = 60, 210, 80
    x, e, t, b = ce_inputs(41, n, v, d, dtype, bias=True)
    t[5] = -1
    up = rnd(42, n) if reduction == "none" else torch.tensor(0.37, dtype=torch.float64)      # upstream gradients of either sign
    counted = int((t >= 0).sum())
    g = up if reduction == "none" else torch.full((n,), 0.37 / (counted if reduction == "mean" else 1), dtype=torch.float64)
    ref = ce_reference(x, e, t, 5.0, b, g)
    tol = ce_tolerances(ref, dtype, n, v, d)
    # a row's gradient enters relative to the largest: one more rounding in float32
    for need in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        xs, es, bs = (a.cuda().requires_grad_(bool(r)) for a, r in zip((x, e, b), need))
        loss = hw.catalogue_cross_entropy(xs, es, t.cuda(), scale=5.0, bias=bs, reduction=reduction)
        loss.backward(up.float().cuda())
        for got, key, r in ((xs.grad, "dx", need[0]), (es.grad, "de", need[1]), (bs.grad, "db", need[2])):
            assert (got is not None) == bool(r)
            if r:
                close(got, ref[key], 1.01 * tol[key] + ref[key + "_size"] * 4 * U32, key)


@gpu
def test_cross_entropy_gradient_against_differences(hw):
    """float32: the gradients along random directions against differences of the 64-bit loss"""
    n, v, d = 30, 77, 40
    x, e, t, b = ce_inputs(51, n, v, d, torch.float32, bias=True)
    loss, dx, de, db = hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), t.cuda(), scale=4.0, bias=b.cuda())
    f = lambda a, c, k: ce_reference(a, c, t, 4.0, k, torch.zeros(n, dtype=torch.float64))["rows"].mean()  # noqa: E731
    s = 1e-5
    for i, got in enumerate((dx, de, db)):
        args = [x.double(), e.double(), b.double()]
        for seed in range(3):
            v_ = rnd(60 + seed, *args[i].shape)
            hi, lo = list(args), list(args)
            hi[i], lo[i] = args[i] + s * v_, args[i] - s * v_
            want = float(f(*hi) - f(*lo)) / (2 * s)
            # the difference's own error is about s^2; every gradient's is within the tolerances above, far below 1e-4 of the sum of magnitudes
            assert abs(float((got.cpu().double() * v_).sum()) - want) <= 1e-4 * float((got.cpu().double() * v_).abs().sum()) / math.sqrt(v_.numel()) + 1e-8


@gpu
def test_cross_entropy_is_the_same_every_time(hw):
    x, e, t, b = (None if a is None else a.cuda() for a in ce_inputs(71, 500, 3000, 128, torch.bfloat16, bias=True))
    first = hw.catalogue_cross_entropy_grads(x, e, t, scale=5.0, bias=b)
    for _ in range(5):
        assert all(torch.equal(p, q) for p, q in zip(first, hw.catalogue_cross_entropy_grads(x, e, t, scale=5.0, bias=b)))


# ---------------------------------------------------------------------------------------------------------------- offsets beyond 32 bits
@gpu
def test_rows_beyond_32_bits(hw):
    """the last rows of operands and outputs of more than 2^32 bytes (and elements): the same as those rows by themselves"""
    free = torch.cuda.mem_get_info()[0]
    if free < 60 << 30:
        pytest.skip("60 GB of device memory needed, %d GB free" % (free >> 30))
    n, d = (1 << 21) + 5, 1024
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(n, d, device="cuda", dtype=torch.bfloat16, generator=g)
    w = torch.randn(d, device="cuda", generator=g)
    last = slice(n - 7, n)
    y, h = hw.rms_norm(x, w, x)
    want = hw.rms_norm(x[last].contiguous(), w, x[last].contiguous())
    assert torch.equal(y[last], want[0]) and torch.equal(h[last], want[1])
    dx, _ = hw.rms_norm_grads(y, h, w)
    assert torch.equal(dx[last], hw.rms_norm_grads(y[last].contiguous(), h[last].contiguous(), w)[0])
    del y, h, dx
    q, s = hw.quantize_rows_q8(x)
    qw, sw = hw.quantize_rows_q8(x[last].contiguous())
    assert torch.equal(q[last], qw) and torch.equal(s[last], sw)
    del x, q, s
    # products: an output, and an operand
    m, k = 66001, 64
    a, b = (torch.randint(-127, 128, (m, k), device="cuda", dtype=torch.int8, generator=g) for _ in range(2))
    one = torch.ones(m, device="cuda")
    out = hw.matmul_q8(a, one, b, one, out_dtype=torch.bfloat16)
    assert out.numel() > 1 << 32 and torch.equal(out[-200:, -200:], (a[-200:].double() @ b[-200:].double().t()).bfloat16())
    del out
    rows = 68_000_003
    tall = torch.randint(-127, 128, (rows, k), device="cuda", dtype=torch.int8, generator=g)
    one = torch.ones(rows, device="cuda")
    for few in (3, 40):
        out = hw.matmul_q8(tall, one, b[:few].contiguous(), one[:few], out_dtype=torch.bfloat16)
        assert torch.equal(out[-100:], (tall[-100:].double() @ b[:few].double().t()).bfloat16())
    out = hw.matmul_q8(b[:2].contiguous(), one[:2], tall, one)
    assert torch.equal(out[:, -100:].double(), b[:2].double() @ tall[-100:].double().t())
    del tall, out, one
    # a catalogue of equal blocks: p is a block's, divided by their number
    block, copies, n, d = 1 << 20, 17, 40, 128
    e = torch.randn(block, d, device="cuda", dtype=torch.bfloat16, generator=g) / 8
    table = e.repeat(copies, 1)
    x = torch.randn(n, d, device="cuda", dtype=torch.bfloat16, generator=g) / 8
    t = torch.randint(0, block, (n,), device="cuda", generator=g)
    assert table.numel() * 2 > 1 << 32
    far = t + (copies - 1) * block
    got = hw.catalogue_cross_entropy(x, table, far, scale=4.0, reduction="none")
    z = 4.0 * (x.double() @ e.double().t())
    want = torch.logsumexp(z, 1) + math.log(copies) - z.gather(1, t[:, None])[:, 0]
    close(got, want.cpu(), (2 * 30 * 8 * math.sqrt(3 * d) + 8 * math.sqrt(block * copies)) * U32, "rows")
    loss, dx, de = hw.catalogue_cross_entropy_grads(x, table, far, scale=4.0)
    # (a float32 sum of 17.8 M terms: 8 sqrt(v) 2^-24 = 2e-3 of the magnitudes, half of which is allowed beside the weights' roundings)
    p = torch.softmax(z, 1)
    dw = 4.0 / n * (p @ e.double() - e[t].double())
    close(dx, dw.cpu(), dw.abs().cpu() * U[torch.bfloat16] + 4.0 / n * ((p @ e.double().abs()) * (U[torch.bfloat16] + 1e-3) + e[t].double().abs() * 1e-3).cpu(), "dx")
    other = torch.ones(block, dtype=torch.bool, device="cuda")
    other[t] = False
    assert torch.equal(de[:block][other], de[-block:][other])
    want = 4.0 / n * (p[:, t].t() @ x.double() / copies - torch.eye(n, device="cuda", dtype=torch.double) @ x.double())
    if len(t.unique()) == n:
        close(de[far], want.cpu(), want.abs().cpu() * U[torch.bfloat16] * 2 + 4.0 / n * x.double().abs().cpu() * 1e-3, "de")


# ---------------------------------------------------------------------------------------------------------------- together, streams, graphs
def _train_and_serve(hw, x, res, w, table, t):
    y, h = hw.rms_norm(x, w, res)
    loss, dy, dtable = hw.catalogue_cross_entropy_grads(y, table, t, scale=0.2)
    dx, dw = hw.rms_norm_grads(dy, h, w)
    q, s, _ = hw.rms_norm_q8(x, w, res)
    cq, cs = hw.quantize_rows_q8(table)
    scores = hw.matmul_q8(q, s, cq, cs)
    return loss, dx, dw, dtable, scores


@gpu
def test_the_operators_together(hw):
    """a training step's gradients through norm and loss, and the scores served in 8 bits, against the 64-bit chain"""
    n, v, d = 100, 400, 64
    x, res = rnd(1, n, d).float(), rnd(2, n, d).float()
    w, table = (1 + 0.1 * rnd(3, d)).float(), (0.3 * rnd(4, v, d)).float()
    t = torch.from_numpy(np.random.default_rng(5).integers(0, v, n))
    loss, dx, dw, dtable, scores = _train_and_serve(hw, *(a.cuda() for a in (x, res, w, table, t)))
    X, W, T = x.double().requires_grad_(), w.double().requires_grad_(), table.double().requires_grad_()
    H = (x + res).double() + (X - X.detach())
    Y, _ = norm_reference(H, W, 1e-6)
    ref = torch.nn.functional.cross_entropy(0.2 * Y @ T.t(), t)
    ref.backward()
    ref = float(ref.detach())
    assert abs(float(loss) - ref) <= 1e-5 * ref
    for got, want in ((dx, X.grad), (dw, W.grad), (dtable, T.grad)):
        assert float((got.cpu().double() - want).norm()) <= 1e-5 * float(want.norm())
    # two factors in 8 bits: half a step of max / 127 each, in every one of the d products
    ys, ts = Y.detach(), table.double()
    step = lambda a: a.abs().amax(1, keepdim=True) / 254  # noqa: E731
    tol = step(ys) * ts.abs().sum(1) + ys.abs().sum(1, keepdim=True) * step(ts).t() + d * step(ys) * step(ts).t()
    close(scores, ys @ ts.t(), 1.001 * tol, "scores")
    # with autograd, through both operators
    xs, ws, tb = x.cuda().requires_grad_(), w.cuda().requires_grad_(), table.cuda().requires_grad_()
    y, h = hw.rms_norm(xs, ws, res.cuda())
    hw.catalogue_cross_entropy(y, tb, t.cuda(), scale=0.2).backward()
    for got, want in ((xs.grad, X.grad), (ws.grad, W.grad), (tb.grad, T.grad)):
        assert float((got.cpu().double() - want).norm()) <= 1e-5 * float(want.norm())


def _chain_inputs(seed, n, v, d, dtype):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    return mk(n, d), mk(n, d), mk(d), mk(v, d), torch.randint(0, v, (n,), generator=g).cuda()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_streams_and_two_calls_at_once(hw, dtype):
    a, b = _chain_inputs(1, 200, 700, 128, dtype), _chain_inputs(2, 200, 700, 128, dtype)
    want = [_train_and_serve(hw, *a), _train_and_serve(hw, *b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(s1):
            g1 = _train_and_serve(hw, *a)
        with torch.cuda.stream(s2):
            g2 = _train_and_serve(hw, *b)
    torch.cuda.synchronize()
    for got, w in ((g1, want[0]), (g2, want[1])):
        assert all(torch.equal(p, q) for p, q in zip(got, w))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_captured_and_replayed(hw, dtype):
    """two graphs of the chain, replayed in turn with eager work between, on new contents of the same buffers"""
    bufs = [_chain_inputs(3, 90, 500, 96, dtype), _chain_inputs(4, 64, 333, 128, dtype)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in bufs:
            _train_and_serve(hw, *x)
    torch.cuda.current_stream().wait_stream(side)
    for x in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_train_and_serve(hw, *x))
        graphs.append(g)
    for turn in range(4):
        for k, (x, g, o) in enumerate(zip(bufs, graphs, outs)):
            new = _chain_inputs(100 + 10 * turn + k, x[0].shape[0], x[3].shape[0], x[0].shape[1], dtype)
            for dst, src in zip(x, new):
                dst.copy_(src)
            g.replay()
            eager = _train_and_serve(hw, *new)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(o, eager)), (turn, k)


@gpu
def test_a_captured_autograd_step(hw):
    """forward and backward through autograd inside a graph, beside eager steps of other leaves"""
    x, res, w, table, t = _chain_inputs(7, 80, 300, 64, torch.float32)

    def step(leaves):
        for p in leaves:
            p.grad = None
        y, _ = hw.rms_norm(leaves[0], leaves[1], res)
        loss = hw.catalogue_cross_entropy(y, leaves[2], t, scale=0.2)
        return (loss.detach(),) + torch.autograd.grad(loss, leaves)
    mine = [p.clone().requires_grad_() for p in (x, w, table)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(mine)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(mine)
    other = [p.clone().requires_grad_() for p in (x, w, table)]
    for turn in range(3):
        with torch.no_grad():
            for a, b in zip(mine, other):
                new = torch.randn_like(a)
                a.copy_(new)
                b.copy_(new)
        g.replay()
        want = step(other)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), turn
