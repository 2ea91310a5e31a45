"""The learned head's operators (hwer/head.py) at the edges of what a call may hold: sizes beyond 32 bits, arguments of other kinds, derivatives that
are not offered, values at the ends of a type's range, many rows.  Tolerances as in test_head.py, whose plain implementations are used."""
import ctypes
import math

import pytest
import torch

from test_head import TINY, TYPES, U, U32, ce_inputs, ce_reference, ce_tolerances, close, codes_reference, gpu, norm_reference, rnd


@pytest.fixture(scope="module")
def hw():
    import hwer
    from hwer import native
    native.lib()
    return hwer


# ---------------------------------------------------------------------------------------------------------------- refusals (no GPU)
WRAPS = [(1 << 32) + 8, (1 << 31) - (1 << 14) + 1, (1 << 31) - 1, 1 << 31, 1 << 40]


@pytest.mark.parametrize("d", WRAPS)
def test_widths_beyond_32_bits_are_refused(hw, d):
    """a width that 32 bits cut off to 8, and those near 2^31 whose columns the wide kernels would count past it (no rows, or addresses that are never read)"""
    from hwer import native
    lib, p, E = native.lib(), ctypes.c_void_p(4096), native.HWER_EINVAL
    for n in (0, 2):
        assert lib.hwer_rms_norm(p, d, None, 0, None, 0, n, d, 0, 1e-6, p, d, None, 0, None) == E
        assert lib.hwer_rms_norm_q8(p, d, None, 0, None, 0, n, d, 0, 1, 1e-6, p, d, p, None, 0, None) == E
        assert lib.hwer_rms_norm_backward(p, d, p, d, None, 0, None, 0, n, d, 0, 1e-6, p, d, None, None, 0, None) == E
    assert lib.hwer_rms_norm_backward_workspace_bytes(2, d) == 16
    for m in (0, 2):
        assert lib.hwer_matmul_q8(p, d, p, p, d, p, None, m, 2, d, p, 2, 0, None) == E
        assert lib.hwer_catalogue_ce(p, d, p, d, None, p, m, 3, d, 0, 1.0, 1, p, p, p, p, None, p, 1 << 50, None) == E
    assert lib.hwer_catalogue_ce_workspace_bytes(2, 3, d, 0, 0, 0, 1) == 0 and lib.hwer_catalogue_ce_reads_in_place(p, d, d, 1) == 0
    # in Python, before anything of that size is allocated (one element that is broadcast)
    x, q, s = torch.zeros(1, 1).expand(2, d), torch.zeros(1, 1, dtype=torch.int8).expand(2, d), torch.zeros(2)
    for f in (lambda: hw.rms_norm(x), lambda: hw.rms_norm_grads(x, x), lambda: hw.rms_norm_q8(x), lambda: hw.quantize_rows_q8(x)):
        with pytest.raises(ValueError, match="at most"):
            f()
    with pytest.raises(native.HwerNativeError):
        hw.matmul_q8(q, s, q, s)      # (host tensors)


@gpu
def test_rows_of_too_many_codes_are_refused(hw):
    for k in (131072, (1 << 32) + 16):
        q, s = torch.zeros(1, 1, dtype=torch.int8, device="cuda").expand(2, k), torch.zeros(2, device="cuda")
        with pytest.raises(ValueError, match="131071 codes"):
            hw.matmul_q8(q, s, q, s)


def test_more_rows_than_a_launch_has_threads_for_are_refused(hw):
    """before anything is launched (these calls used to fail at a later launch; the addresses are never read)"""
    from hwer import native
    lib, p, E = native.lib(), ctypes.c_void_p(4096), native.HWER_EINVAL
    for n in ((1 << 26) - 255, 1 << 26, 1 << 30):
        assert lib.hwer_catalogue_ce(p, 8, p, 8, None, p, n, 3, 8, 0, 1.0, 1, p, p, p, p, None, p, 1 << 50, None) == E
        assert lib.hwer_catalogue_ce_grads(p, 8, p, 8, None, p, n, 3, 8, 0, 1.0, 1, p, p, 8, p, 8, None, p, 1 << 50, None) == E
        assert lib.hwer_catalogue_ce_workspace_bytes(n, 3, 8, 0, 0, 0, 1) == 0 and lib.hwer_catalogue_ce_workspace_bytes(3, 64 * n, 8, 0, 0, 0, 1) == 0
        assert lib.hwer_catalogue_ce_backward(p, 8, p, 8, None, p, n, 3, 8, 0, 1.0, 1, p, p, p, p, p, 8, p, 8, None, p, 1 << 50, None) == E
    for m, n, k in ((1, 1 << 30, 16), (1 << 30, 32, 512), (1 << 28, 5, 513), (40, (1 << 31) - 256, 64), (1 << 30, 1 << 30, 8), (1 << 31, 2, 8)):
        assert lib.hwer_matmul_q8(p, k, p, p, k, p, None, m, n, k, p, n, 0, None) == E, (m, n, k)


def test_workspaces_off_their_alignment_are_refused(hw):
    from hwer import native
    lib, p, E = native.lib(), ctypes.c_void_p(4096), native.HWER_EINVAL
    at = lambda off: ctypes.c_void_p(4096 + off)  # noqa: E731
    for off in (1, 4, 16, 128):
        assert lib.hwer_catalogue_ce(p, 8, p, 8, None, p, 2, 3, 8, 0, 1.0, 1, p, p, p, p, None, at(off), 1 << 40, None) == E
        assert lib.hwer_catalogue_ce_grads(p, 8, p, 8, None, p, 2, 3, 8, 0, 1.0, 1, p, p, 8, p, 8, None, at(off), 1 << 40, None) == E
        assert lib.hwer_catalogue_ce_backward(p, 8, p, 8, None, p, 2, 3, 8, 0, 1.0, 1, p, p, p, p, p, 8, p, 8, None, at(off), 1 << 40, None) == E
    for off in (1, 4, 8):
        assert lib.hwer_catalogue_ce(p, 8, p, 8, None, p, 2, 3, 8, 0, 1.0, 1, p, at(off), p, p, None, p, 1 << 40, None) == E
        assert lib.hwer_catalogue_ce_backward(p, 8, p, 8, None, p, 2, 3, 8, 0, 1.0, 1, p, at(off), p, p, p, 8, p, 8, None, p, 1 << 40, None) == E
        assert lib.hwer_rms_norm_backward(p, 8, p, 8, p, 0, None, 0, 2, 8, 0, 1e-6, p, 8, p, at(off), 1 << 40, None) == E


def test_dual_tensors_are_refused(hw):
    """a forward-mode tangent would be lost without a word: requires_grad is False on a dual tensor"""
    import torch.autograd.forward_ad as fw
    x, w, t, q, s = torch.ones(3, 8), torch.ones(8), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 8, dtype=torch.int8), torch.ones(3)
    with fw.dual_level():
        dual = lambda a: fw.make_dual(a, torch.ones_like(a))  # noqa: E731
        for f in (lambda: hw.rms_norm(dual(x)), lambda: hw.rms_norm(x, dual(w)), lambda: hw.rms_norm(x, w, dual(x)), lambda: hw.rms_norm_grads(dual(x), x),
                  lambda: hw.rms_norm_grads(x, x, dh=dual(x)), lambda: hw.rms_norm_q8(dual(x)), lambda: hw.quantize_rows_q8(dual(x)), lambda: hw.matmul_q8(q, dual(s), q, s),
                  lambda: hw.matmul_q8(q, s, q, s, bias=dual(s)), lambda: hw.catalogue_cross_entropy(dual(x), x, t), lambda: hw.catalogue_cross_entropy(x, dual(x), t),
                  lambda: hw.catalogue_cross_entropy(x, x, t, bias=dual(s)), lambda: hw.catalogue_cross_entropy_grads(dual(x), x, t)):
            with pytest.raises(NotImplementedError):
                f()
        with pytest.raises(Exception):      # (beside a leaf torch's own refusal may come first)
            hw.rms_norm(dual(x), torch.ones(8, requires_grad=True))
        from hwer import native
        with pytest.raises(native.HwerNativeError):      # no dual among the operands: as ever (these are on the host)
            hw.rms_norm(x)


def test_profiles_of_the_search_are_bound_to_the_search():
    """the digest that the search's traffic counters carry covers every file that its kernels include, and none of the learned head's"""
    import os
    import re
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    csrc = os.path.join(root, "hybrid-weighted-embedding-recommender_amd", "csrc")
    sys.path.insert(0, csrc)
    try:
        import build as hip_build
    finally:
        sys.path.pop(0)
    mine = set(hip_build.SEARCH_SOURCES + hip_build.SEARCH_HEADERS)
    assert not {f for f in mine if "head_" in f or "catalogue" in f or "q8" in f} and set(hip_build.SEARCH_SOURCES) < set(hip_build.SOURCES)
    for f in mine:
        with open(os.path.join(csrc, f)) as fh:
            for inc in re.findall(r'#include "([^"]+)"', fh.read()):
                assert inc in mine or inc == "hwer_hip.h", (f, inc)
    assert hip_build.search_digest() not in (hip_build._digest(), hip_build._digest(hip_build.SEARCH_SOURCES))


def test_a_learned_scale_is_refused(hw):
    """its gradient would be lost without a word"""
    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    scale = torch.tensor(20.0, requires_grad=True)
    with pytest.raises(NotImplementedError, match="queries"):
        hw.catalogue_cross_entropy(x, x, t, scale=scale)
    from hwer import native
    for other in (scale.detach(), 20):
        with pytest.raises(native.HwerNativeError):      # (host tensors)
            hw.catalogue_cross_entropy(x, x, t, scale=other)
    with torch.no_grad(), pytest.raises(native.HwerNativeError):
        hw.catalogue_cross_entropy(x, x, t, scale=scale)


# ---------------------------------------------------------------------------------------------------------------- what a call may be given (GPU)
@gpu
def test_operators_without_a_gradient_say_so(hw):
    x, w, q, s = torch.ones(3, 8, device="cuda"), torch.ones(8, device="cuda"), torch.zeros(3, 8, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")
    p = lambda a: a.clone().requires_grad_()  # noqa: E731
    calls = (lambda: hw.rms_norm_q8(p(x)), lambda: hw.rms_norm_q8(x, p(w)), lambda: hw.rms_norm_q8(x, w, p(x)), lambda: hw.quantize_rows_q8(p(x)), lambda: hw.matmul_q8(q, p(s), q, s),
             lambda: hw.matmul_q8(q, s, q, p(s)), lambda: hw.matmul_q8(q, s, q, s, bias=p(s)))
    for f in calls:
        with pytest.raises(NotImplementedError, match="no_grad"):
            f()
        with torch.no_grad():
            f()
    # the gradients' own functions take parameters as they are
    assert hw.rms_norm_grads(x, x, p(w))[1].shape == (8,) and hw.catalogue_cross_entropy_grads(p(x), p(x), torch.zeros(3, dtype=torch.int64, device="cuda"))[1].shape == (3, 8)


@gpu
def test_operands_that_are_no_tensors_raise_type_errors(hw):
    x, w, q, s, t = torch.ones(3, 8, device="cuda"), torch.ones(8, device="cuda"), torch.zeros(3, 8, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in ([1.0] * 8, 1.0, w.cpu().numpy()):
        for f in (lambda: hw.rms_norm(bad), lambda: hw.rms_norm(x, bad), lambda: hw.rms_norm(x, w, bad), lambda: hw.rms_norm_grads(bad, x), lambda: hw.rms_norm_grads(x, bad),
                  lambda: hw.rms_norm_grads(x, x, bad), lambda: hw.rms_norm_grads(x, x, dh=bad), lambda: hw.rms_norm_q8(x, bad), lambda: hw.rms_norm_q8(x, w, bad),
                  lambda: hw.quantize_rows_q8(bad), lambda: hw.matmul_q8(bad, s, q, s), lambda: hw.matmul_q8(q, bad, q, s), lambda: hw.matmul_q8(q, s, q, bad),
                  lambda: hw.matmul_q8(q, s, q, s, bias=bad), lambda: hw.catalogue_cross_entropy(bad, x, t), lambda: hw.catalogue_cross_entropy(x, bad, t),
                  lambda: hw.catalogue_cross_entropy(x, x, bad), lambda: hw.catalogue_cross_entropy(x, x, t, bias=bad), lambda: hw.catalogue_cross_entropy_grads(x, x, bad)):
            with pytest.raises(TypeError):
                f()
    for f in (lambda: hw.rms_norm_grads(None, x), lambda: hw.matmul_q8(q, None, q, s), lambda: hw.matmul_q8(q, s, q, None), lambda: hw.catalogue_cross_entropy(x, x, None)):
        with pytest.raises(TypeError):
            f()


# ---------------------------------------------------------------------------------------------------------------- codes
def exact_codes(h, w):
    """round_half_even(127 v / max|v|) of one row in integers (values as fractions)"""
    from fractions import Fraction
    v = [Fraction(float(a)) * Fraction(float(b)) for a, b in zip(h, w)]
    top = max(abs(a) for a in v)
    return torch.tensor([round(127 * a / top) for a in v], dtype=torch.int8)      # (Python rounds fractions to even)


# 24-bit factors h, w and H, W of a row's largest product, whose quotient 127 h w / (H W) misses a border between two codes by about 2^-52 of itself
NEAR_BORDERS = [(9421653, 11442761, 11141540, 15856770), (11326493, 15955928, 14549902, 14674142)]


@gpu
@pytest.mark.parametrize("d", [4, 24, 1000, 4096, 40961])
def test_q8_codes_next_to_a_border_are_exact(hw, d):
    for h, w, top_h, top_w in NEAR_BORDERS:
        for near in (0, 1, -1):      # beside it: the same product one step of a factor further
            x, y = torch.zeros(2, d), torch.ones(d)
            x[0, :4] = torch.tensor([float(top_h), float(h), -float(h), float(h + near)])
            y[:4] = torch.tensor([float(top_w), float(w), float(w), float(w)])
            x[1] = 0.5 * x[0]
            want = exact_codes(x[0], y)
            q = hw.rms_norm_q8(x.cuda(), y.cuda())[0].cpu()
            assert torch.equal(q[0], want) and torch.equal(q[1], want), (q[:, :4], want[:4])


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("d", [9, 24, 250, 4096, 40961])
def test_q8_codes_of_the_largest_values_are_exact(hw, d, dtype):
    """rows that reach 127 * 2^121, whose 127-fold is beyond float32: values on the borders between two codes, and next to them"""
    steps = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 3.5, 100.5, -126.5])
    x = torch.zeros(2, d, dtype=torch.float64)
    x[0, :9], x[0, 9:] = steps, 50 * torch.tanh(rnd(d, d - 9))
    x[1, :9] = -steps
    x = (x * 2.0 ** 121).to(dtype)
    if dtype == torch.float32 and d > 9:
        x[:, 9] = torch.nextafter(x[:, 7], x[:, 0])      # 100.5 and -100.5, one step of float32 upwards / away
        x[:, 10] = torch.nextafter(x[:, 8], x[:, 0])
    codes, top = codes_reference(x, None)
    q, s = hw.quantize_rows_q8(x.cuda())
    assert torch.equal(q.cpu(), codes)
    close(s, top / 127, top / 127 * 3 * U32, "scale")
    # the same as products: rows of 2^41 (their squares are in range) and weights of 2^80
    for w in (torch.full((d,), 2.0 ** 80), torch.full((d,), 2.0 ** 80).to(dtype)):
        q, s = hw.rms_norm_q8((x.double() * 2.0 ** -80).to(dtype).cuda(), w.cuda())
        assert torch.equal(q.cpu(), codes)

@gpu
@pytest.mark.parametrize("d", [24, 4096, 40961])
def test_q8_scale_of_a_row_of_zeros_is_zero(hw, d):
    """... whatever eps is: without one its norm is 0 / 0, but the codes' scale is not"""
    x = torch.zeros(3, d)
    x[1, 2] = 1.0
    for w in (None, torch.ones(d).cuda(), torch.zeros(d).cuda()):
        q, s = hw.rms_norm_q8(x.cuda(), w, eps=0.0)
        assert float(s[0]) == 0 and float(s[2]) == 0 and not q[0].any() and not q[2].any() and torch.isfinite(s).all()


# ---------------------------------------------------------------------------------------------------------------- strides
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,d", [(1, 7), (9, 100), (130, 250), (33, 1024), (5, 4100), (3, 20001)])
def test_norm_of_strided_operands(hw, n, d, dtype):
    """every operand as rows of a wider tensor (at any alignment), transposed, broadcast and with a leading dimension: the same bits as of copies"""
    x, res, dy, dh = (rnd(n + i, n, d).to(dtype).cuda() for i in range(4))
    w = (1 + 0.2 * rnd(9, d)).to(dtype).cuda()

    def wide(t, left):
        out = torch.full((n, d + 13), float("nan"), dtype=dtype, device="cuda")
        out[:, left:left + d] = t
        return out[:, left:left + d]
    views = {"wide": lambda t, i: wide(t, 1 + 2 * i), "transposed": lambda t, i: t.t().contiguous().t(), "leading": lambda t, i: wide(t, i).unsqueeze(1),
             "every second": lambda t, i: torch.stack([t, t], -1).reshape(n, 2 * d)[:, ::2]}
    weights = torch.stack([w, w], 1).reshape(-1)[::2]
    y, h = hw.rms_norm(x, w, res)
    dx, dw = hw.rms_norm_grads(dy, h, w, dh=dh)
    q, s, hq = hw.rms_norm_q8(x, w, res)
    plain, scale = hw.quantize_rows_q8(x)
    for name, view in views.items():
        vx, vr, vy, vd, vh = (view(t, i) for i, t in enumerate((x, res, dy, dh, h)))
        got = (hw.rms_norm(vx, weights, vr), hw.rms_norm_grads(vy, vh, weights, dh=vd), hw.rms_norm_q8(vx, weights, vr), hw.quantize_rows_q8(vx))
        for out, want in zip(got, ((y, h), (dx, dw), (q, s, hq), (plain, scale))):
            assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(out, want)), name
        leaves = [t.detach().requires_grad_() for t in (vx, weights, vr)]
        out, hidden = hw.rms_norm(leaves[0], leaves[1], leaves[2])
        torch.autograd.backward([out, hidden], [vy, vd])
        assert torch.equal(leaves[0].grad.reshape(n, d), dx) and torch.equal(leaves[2].grad.reshape(n, d), dx) and torch.equal(leaves[1].grad, dw), name
    # one row for all, and one gradient for all
    row = x[:1].expand(n, d)
    assert torch.equal(hw.rms_norm(row, w, res)[0], hw.rms_norm(row.contiguous(), w, res)[0]) and torch.equal(hw.rms_norm_q8(row, w)[0], hw.rms_norm_q8(row.contiguous(), w)[0])
    assert torch.equal(hw.rms_norm_grads(dy[:1].expand(n, d), h, w)[0], hw.rms_norm_grads(dy[:1].expand(n, d).contiguous(), h, w)[0])
    z = x.clone().requires_grad_()
    hw.rms_norm(z, w).sum().backward()
    assert torch.equal(z.grad, hw.rms_norm_grads(torch.ones_like(x), x, w)[0])


# ---------------------------------------------------------------------------------------------------------------- cross entropy
@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(40, 333, 64), (70, 150, 100), (300, 90, 256)])
def test_cross_entropy_of_a_target_that_is_taken_out(hw, n, v, d, dtype):
    """its row's loss is infinite; whatever the class holds reaches no gradient, and it has none itself"""
    x, e, t, b = ce_inputs(n + d, n, v, d, dtype, bias=True)
    b[3::7] = float("-inf")
    t[::4] = 3
    t[1::4] = 10
    t[2] = -1
    gone = torch.isinf(b)
    bad, clean = e.clone(), e.clone()
    clean[gone] = 0
    bad[gone] = float("nan")
    bad[10], bad[17] = float("inf"), torch.finfo(dtype).max
    out_of = gone[t.clamp_min(0)] & (t >= 0)
    # a class of its own, at -inf, that the target names: neither its row nor its gradients are of the table
    ref_e, ref_b, ref_t = torch.cat([clean, torch.zeros(1, d, dtype=dtype)]), torch.cat([b, b[3:4]]), torch.where(out_of, torch.tensor(v), t)
    up = torch.linspace(-1, 1, n).double()
    up[out_of & (torch.arange(n) % 8 < 4)] = 0          # the caller drops some of the infinite losses
    counted = int((t >= 0).sum())
    one = torch.full((n,), 1.0 / counted, dtype=torch.float64)
    for form, g in (("grads", one), ("mean", one), ("none", up)):
        ref = ce_reference(x, ref_e, ref_t, 4.0, ref_b, g)
        tol = ce_tolerances(ref, dtype, n, v, d)
        if form == "grads":
            loss, dx, de, db = hw.catalogue_cross_entropy_grads(x.cuda(), bad.cuda(), t.cuda(), scale=4.0, bias=b.cuda())
        else:
            leaves = [a.cuda().requires_grad_() for a in (x, bad, b)]
            loss = hw.catalogue_cross_entropy(leaves[0], leaves[1], t.cuda(), scale=4.0, bias=leaves[2], reduction=form)
            loss.backward(None if form == "mean" else up.float().cuda())
            dx, de, db = (a.grad for a in leaves)
        if form == "none":
            assert torch.isinf(loss.detach().cpu()[out_of]).all() and torch.isfinite(loss.detach().cpu()[~out_of]).all()
        else:
            assert float(loss.detach()) == float("inf")
        for got, key in ((dx, "dx"), (de, "de"), (db, "db")):
            close(got, ref[key] if key == "dx" else ref[key][:v], 1.01 * (tol[key] if key == "dx" else tol[key][:v]) + (ref[key + "_size"] * 4 * U32)[:v if key != "dx" else n], form + " " + key)
        assert not de[gone.cuda()].any() and not db[gone.cuda()].any()


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(2049, 300, 64), (5000, 129, 128), (8192, 40, 32), (8193, 40, 32), (16384, 33, 20), (16385, 33, 20), (20000, 300, 64), (70001, 17, 130)])
def test_cross_entropy_of_many_rows(hw, n, v, d, dtype):
    """counts, losses and the largest upstream gradient of more rows than a wave's lanes, a row's share and a workgroup's, in each form; the same every time"""
    x, e, t, _ = ce_inputs(n + v, n, v, d, dtype)
    t[::5] = -1
    t[n - 1] = 1
    counted = int((t >= 0).sum())
    dev = [a.cuda() for a in (x, e, t)]
    up = rnd(7, n)
    up[::4] = 0
    up[n - 2] = 9.0                  # the largest one, among the last rows
    t64 = [a.cuda() for a in (x, e, t)]
    for form, g in (("mean", torch.full((n,), 1.0 / counted, dtype=torch.float64)), ("sum", torch.ones(n, dtype=torch.float64)), ("none", up)):
        ref = {k: a.cpu() for k, a in ce_reference(t64[0], t64[1], t64[2], 4.0, None, g.cuda()).items()}
        tol = ce_tolerances(ref, dtype, n, v, d)
        low = 0.0 if dtype == torch.bfloat16 or form != "none" else 2.0 ** -40 * 4.0 * up.abs().max() * x.double().abs().sum(0)
        want = ref["rows"].sum() / (counted if form == "mean" else 1)
        if form != "none":
            out = hw.catalogue_cross_entropy_grads(*dev, scale=4.0, reduction=form)
            close(out[0], want, tol["loss"] * (1 if form == "mean" else n) + want.abs() * 2 * U32, form + " loss")
            close(out[1], ref["dx"], tol["dx"], form + " dqueries")
            close(out[2], ref["de"], tol["de"], form + " dtable")
            assert all(torch.equal(p, q) for p, q in zip(out, hw.catalogue_cross_entropy_grads(*dev, scale=4.0, reduction=form)))
        q, tab = dev[0].clone().requires_grad_(), dev[1].clone().requires_grad_()
        loss = hw.catalogue_cross_entropy(q, tab, dev[2], scale=4.0, reduction=form)
        if form == "none":
            close(loss, ref["rows"], tol["loss"] + ref["rows"].abs() * U32, "rows")
        else:
            assert torch.equal(loss.detach(), out[0])
        loss.backward(up.float().cuda() if form == "none" else None)
        close(q.grad, ref["dx"], 1.01 * tol["dx"] + ref["dx_size"] * 4 * U32, form + " autograd dqueries")
        close(tab.grad, ref["de"], 1.01 * tol["de"] + ref["de_size"] * 4 * U32 + low, form + " autograd dtable")


def equal_rows(n, v, d, dtype, bias):
    """Four kinds of queries over a catalogue of one row again and again, one that is a little better and one that is far off (the target of most): every
    weight of a long sum is the same value, so that its roundings have one direction.  Products of rows are exact in every type (a few bits each).
    -> operands on the device, and the 64-bit results"""
    a = torch.tensor([1.0, 0.5, 0.25, 0.75]).repeat(d // 4).to(dtype).cuda()
    unit = torch.tensor([2.0, 4.0, 0.0, 0.0]).repeat(d // 4).to(dtype).cuda() / d          # <unit, a> = 1
    table = a.repeat(v, 1)
    table[0] = a * 1.25          # (the first one, so that the others' weights are below 1 from the start)
    table[v - 1] = a * -0.25
    kind = torch.arange(n, device="cuda") % 4
    kinds = torch.stack([unit * c for c in (0.875, 1.25, 1.75, 2.875)])
    queries = kinds[kind]
    target = torch.where(torch.arange(n, device="cuda") % 5 == 0, v // 2, v - 1)
    b = None
    if bias:
        b = torch.full((v,), 0.37, device="cuda")
        b[v // 5] = -1.0
    z = kinds.double() @ table.double().t() + (0 if b is None else b.double())
    lse = torch.logsumexp(z, 1)
    p = torch.exp(z - lse[:, None])
    rows = lse[kind] - z[kind, target]
    mean = p @ table.double()
    dx = (mean[kind] - table[target].double()) / n
    dx_size = (p @ table.double().abs())[kind] / n + table[target].double().abs() / n
    w, wa = torch.zeros_like(p), torch.zeros_like(p)
    for k in range(4):
        hot = torch.zeros(v, dtype=torch.float64, device="cuda")
        for c in (v // 2, v - 1):
            hot[c] = int(((kind == k) & (target == c)).sum())
        w[k], wa[k] = (p[k] * int((kind == k).sum()) - hot) / n, (p[k] * int((kind == k).sum()) + hot) / n
    de, de_size = w.t() @ kinds.double(), wa.t() @ kinds.double().abs()
    return (queries, table, target, b), dict(rows=rows, dx=dx, dx_size=dx_size, de=de, de_size=de_size, db=w.sum(0), db_size=wa.sum(0))


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,v,bias", [(65536, 1200001, False), (4096, 1200001, True), (1200001, 65536, True), (512, 2500000, False)])
def test_cross_entropy_sums_over_long_catalogues_and_batches(hw, n, v, bias, dtype):
    """float32 sums of a million equal terms.  The sums of probabilities are compensated: off by a few roundings, whatever their length.  The products'
    sums are added by the matrix instructions, at most 1 536 (float32 rows) or 8 192 of them one after the other: each rounding is up to 2^-24 of a sum that is
    half of the last one on the average, so N of one direction leave up to N 2^-25; and joined from up to 512 parts, which may leave 512 2^-25 more."""
    d = 64
    (x, e, t, b), ref = equal_rows(n, v, d, dtype, bias)
    f32 = dtype == torch.float32
    # a logit of |z| < 4 in powers of two: the factor's and the product's rounding, and that of a sum below 16; a probability: two of them, and the
    # exponential's and the sums' few roundings
    dz = 4 * 2 * U32 + 2.0 ** -21
    dp = 2 * dz + 16 * U32
    rows = hw.catalogue_cross_entropy(x, e, t, bias=b, reduction="none")
    close(rows, ref["rows"].cpu(), dz + 16 * U32 + ref["rows"].cpu().abs() * U32, "rows")
    out = hw.catalogue_cross_entropy_grads(x, e, t, bias=b)
    assert abs(float(out[0]) - float(ref["rows"].mean())) <= dz + 32 * U32
    long = ((1536 if f32 else 8192) + 512) * 2.0 ** -25
    w = 2.0 ** -22 if f32 else U[dtype]
    low = 0.0 if dtype == torch.bfloat16 else 2.0 ** -36 * 4 * float(e.double().abs().amax()) / n
    close(out[1], ref["dx"].cpu(), ref["dx"].cpu().abs() * U[dtype] + ref["dx_size"].cpu() * (dp + long + w) + low + 4 * TINY[dtype], "dqueries")
    floor = 0.0 if dtype == torch.bfloat16 else 2.0 ** -40 * float(x.double().abs().amax())
    close(out[2], ref["de"].cpu(), ref["de"].cpu().abs() * U[dtype] + ref["de_size"].cpu() * (dp + long + w) + floor + 4 * TINY[dtype], "dtable")
    if bias:
        close(out[3], ref["db"].cpu(), ref["db_size"].cpu() * (dp + 512 * 2.0 ** -25) + 1e-30, "dbias")


@gpu
@pytest.mark.parametrize("n,v,d", [(5, 9, 64), (70, 333, 100), (300, 2000, 128), (40, 150, 256)])
@pytest.mark.parametrize("exponent", [-118, -100, 60, 90, 118])
def test_cross_entropy_of_float32_rows_far_from_one(hw, n, v, d, exponent):
    """queries of size 2^k against rows of size 2^-k: the logits are ordinary, and so are the relative errors of everything"""
    x, e, t, b = ce_inputs(n + d, n, v, d, torch.float32, bias=True)
    x, e = (x.double() * 2.0 ** exponent).float(), (e.double() * 2.0 ** -exponent).float()
    t[::5] = -1
    counted = int((t >= 0).sum())
    for bias in (None, b):
        ref = ce_reference(x, e, t, 5.0, bias, torch.full((n,), 1.0 / counted, dtype=torch.float64))
        tol = ce_tolerances(ref, torch.float32, n, v, d)
        grads = hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), t.cuda(), scale=5.0, bias=None if bias is None else bias.cuda())
        leaves = [None if a is None else a.cuda().requires_grad_() for a in (x, e, bias)]
        loss = hw.catalogue_cross_entropy(leaves[0], leaves[1], t.cuda(), scale=5.0, bias=leaves[2])
        loss.backward()
        for out in (grads, [loss] + [a.grad for a in leaves if a is not None]):
            close(out[0], ref["rows"].sum() / counted, tol["loss"] + ref["rows"].sum().abs() / counted * 2 * U32, "loss")
            for got, key in zip(out[1:], ("dx", "de", "db")):
                # (results below the smallest normal value keep its step)
                close(got, ref[key], 1.01 * (tol[key] - (4 * TINY[torch.float32] if key != "db" else 0)) + ref[key + "_size"] * 4 * U32 + 2.0 ** -148, key)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("n,v,d", [(200, 4000, 64), (1000, 1300, 100), (700, 5000, 128), (300, 900, 256)])
@pytest.mark.parametrize("bias", [False, True])
def test_cross_entropy_gradient_of_a_class_that_is_a_target_once(hw, n, v, d, dtype, bias):
    """its one large weight, the target's, is not rounded to 16 bits: what is left is the rounding of the gradient itself and of the small weights"""
    x, e, _, b = ce_inputs(n + d, n, v, d, dtype, bias=bias, spread=0.0)
    t = torch.randperm(v, generator=torch.Generator().manual_seed(n))[:n]
    t[::9] = -1
    for form in ("mean", "none"):
        up = (0.5 + torch.rand(n, generator=torch.Generator().manual_seed(d))).double() / n if form == "none" else torch.full((n,), 1.0 / int((t >= 0).sum()), dtype=torch.float64)
        ref = ce_reference(x, e, t, 3.0, b, up)
        tol = ce_tolerances(ref, dtype, n, v, d)
        z = 3.0 * (x.double() @ e.double().t()) + (0 if b is None else b.double())
        p = torch.softmax(z, 1) * torch.where(t >= 0, up, torch.zeros_like(up))[:, None]
        hot = torch.zeros_like(p).scatter_(1, t.clamp_min(0)[:, None], 1.0) * torch.where(t >= 0, up, torch.zeros_like(up))[:, None]
        small, large = 3.0 * (p.t() @ x.double().abs()), 3.0 * (hot.t() @ x.double().abs())
        u = U[dtype]
        want = tol["de"] - ref["de_p"] * u + small * u + large * 2 * u * u + ref["de_size"] * 4 * U32
        tab = e.cuda().requires_grad_()
        hw.catalogue_cross_entropy(x.cuda(), tab, t.cuda(), scale=3.0, bias=None if b is None else b.cuda(), reduction=form).backward(up.float().cuda() if form == "none" else None)
        close(tab.grad, ref["de"], want, form + " dtable")
        if form == "mean":
            close(hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), t.cuda(), scale=3.0, bias=None if b is None else b.cuda())[2], ref["de"], want, "dtable in one call")


@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy_of_no_rows_through_autograd(hw, reduction):
    """an empty batch: losses and gradients of a sum over nothing"""
    for dtype in TYPES:
        q, e, b = torch.zeros(0, 40, dtype=dtype, device="cuda").requires_grad_(), rnd(1, 70, 40).to(dtype).cuda().requires_grad_(), rnd(2, 70).float().cuda().requires_grad_()
        loss = hw.catalogue_cross_entropy(q, e, torch.zeros(0, dtype=torch.int64, device="cuda"), bias=b, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and not loss.detach().any()
        loss.backward(torch.zeros(0, device="cuda") if reduction == "none" else None)
        assert q.grad.shape == (0, 40) and not e.grad.any() and not b.grad.any()


@gpu
def test_cross_entropy_of_many_rows_captured(hw):
    """the sums in parts inside two graphs, replayed in turn on new contents, with eager calls between"""
    n, v, d = 20000, 300, 64
    make = lambda seed: tuple(a.cuda() for a in ce_inputs(seed, n, v, d, torch.bfloat16)[:3])  # noqa: E731
    bufs, graphs, outs = [make(1), make(2)], [], []

    def call(x, e, t):
        rows = hw.catalogue_cross_entropy(x, e, t, scale=4.0, reduction="none")
        return (rows,) + tuple(hw.catalogue_cross_entropy_grads(x, e, t, scale=4.0)) + (hw.catalogue_cross_entropy(x, e, t, scale=4.0),)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for b in bufs:
            call(*b)
    torch.cuda.current_stream().wait_stream(side)
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(*b))
        graphs.append(g)
    for turn in range(3):
        for k in (0, 1):
            new = make(10 + 2 * turn + k)
            for dst, src in zip(bufs[k], new):
                dst.copy_(src)
            graphs[k].replay()
            want = call(*new)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs[k], want)), (turn, k)


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("mask", [-1e4, -1.7e7, -4e7, -5e7, -6.5e7, -1e8, -1e9, -1e30])
def test_cross_entropy_of_finite_masks(hw, dtype, mask):
    """classes put far away by a finite offset, whole tiles of them first, with logits that rise: as good as gone, whatever float32's steps are out there"""
    n, v, d, gone = 300, 60000, 64, 40000          # (several tiles to a split)
    x, e, t, b = ce_inputs(77, n, v, d, dtype, bias=True, spread=0.0)
    e[:gone] = (e[:gone].float() * torch.linspace(1, 6, 128).repeat(gone // 128 + 1)[:gone, None]).to(dtype)
    b[:gone] = mask
    t = gone + t % (v - gone)
    kept = torch.arange(v) >= gone
    one = torch.full((n,), 1.0 / n, dtype=torch.float64)
    ref = {k: a.cpu() for k, a in ce_reference(x.cuda(), e.cuda(), t.cuda(), 30.0, torch.where(kept, b, torch.tensor(float("-inf"))).cuda(), one.cuda()).items()}
    tol = ce_tolerances(ref, dtype, n, v, d)
    loss, dx, de, db = hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), t.cuda(), scale=30.0, bias=b.cuda())
    close(loss, ref["rows"].mean(), tol["loss"] + ref["rows"].mean().abs() * 2 * U32, "loss")
    close(dx, ref["dx"], tol["dx"], "dqueries")
    close(de, ref["de"], tol["de"], "dtable")
    close(db, ref["db"], tol["db"], "dbias")


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("mask", [-1e4, -4e7, -1e9, -1e30, -3e38, float(torch.finfo(torch.float32).min)])
@pytest.mark.parametrize("n,v,d", [(60, 90, 64), (300, 2000, 100)])
def test_cross_entropy_of_a_target_at_a_finite_mask(hw, n, v, d, dtype, mask):
    """its loss is as large as the mask, its probability nothing, and everything else as if it were far away"""
    x, e, t, b = ce_inputs(n + d, n, v, d, dtype, bias=True, spread=0.0)
    b[: v // 3] = mask
    t = v // 3 + t % (v - v // 3)
    t[::5] = 7
    t[1::10] = -1
    far = t == 7
    counted = int((t >= 0).sum())
    up = torch.where(t >= 0, 1.0 / counted, 0.0).double()
    ref = ce_reference(x, e, t, 4.0, b, up)
    tol = ce_tolerances(ref, dtype, n, v, d)
    leaves = [a.cuda().requires_grad_() for a in (x, e, b)]
    rows = hw.catalogue_cross_entropy(leaves[0], leaves[1], t.cuda(), scale=4.0, bias=leaves[2], reduction="none")
    # (the target's logit is rounded at the mask's size)
    close(rows, ref["rows"].clamp_max(float(torch.finfo(torch.float32).max)), tol["loss"] + ref["rows"].abs() * U32 + torch.where(far, abs(mask) * 2 * U32, 0.0), "rows")
    rows.backward(up.float().cuda())
    grads = hw.catalogue_cross_entropy_grads(x.cuda(), e.cuda(), t.cuda(), scale=4.0, bias=b.cuda())
    for dx, de, db in (tuple(a.grad for a in leaves), grads[1:]):
        close(dx, ref["dx"], 1.01 * tol["dx"] + ref["dx_size"] * 4 * U32, "dqueries")
        close(de, ref["de"], 1.01 * tol["de"] + ref["de_size"] * 4 * U32, "dtable")
        close(db, ref["db"], 1.01 * tol["db"] + ref["db_size"] * 4 * U32, "dbias")


@gpu
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale", [1e4, 3e6, 1e7, 3e7, 1e8])
@pytest.mark.parametrize("bias", [False, True])
def test_cross_entropy_of_huge_logits(hw, dtype, scale, bias):
    """logits whose float32 steps are beyond one: each row's probability is at one class, and everything stays finite"""
    n, v, d = 200, 700, 64
    x, e, t, _ = ce_inputs(5, n, v, d, dtype, spread=0.0)
    x, e = (x.float() * 2).to(dtype), (e.float() * 2).to(dtype)
    z = x.double() @ e.double().t()
    best = z.topk(2, 1)
    clear = (best.values[:, 0] - best.values[:, 1]) * scale > 200 + 64 * scale * 2.0 ** -22      # (the second class is out of reach)
    t[::3] = best.indices[::3, 0]
    t[~clear] = -1
    assert int((t >= 0).sum()) > n // 2
    up = torch.full((n,), 0.01 / scale, dtype=torch.float64)
    leaves = [a.cuda().requires_grad_() for a in (x, e)]
    b = torch.zeros(v, device="cuda") if bias else None
    rows = hw.catalogue_cross_entropy(leaves[0], leaves[1], t.cuda(), scale=scale, bias=b, reduction="none")
    rows.backward(up.float().cuda())
    on = (t >= 0)
    at = t.clamp_min(0)
    want = torch.where(on, scale * (best.values[:, 0] - z.gather(1, at[:, None])[:, 0]), 0.0)
    size = scale * (x.double().abs() @ e.double().abs().t()).amax(1)
    close(rows, want, size * (9 * 2.0 ** -22 + 40 * U32) + 1e-30, "rows")
    g = (scale * up * on)[:, None]
    top, mine = e.double()[best.indices[:, 0]], e.double()[at]
    u = U[dtype]
    close(leaves[0].grad, g * (top - mine), g * (top.abs() + mine.abs()) * (2 * u + 1e-5) + 4 * TINY[dtype], "dqueries")
    de, de_size = torch.zeros(v, d, dtype=torch.float64), torch.zeros(v, d, dtype=torch.float64)
    for sign, idx in ((1, best.indices[:, 0]), (-1, at)):
        de.index_add_(0, idx, sign * g * x.double())
        de_size.index_add_(0, idx, g * x.double().abs())
    # a probability next to 1 comes from a difference of logits: float32's step there, up to the probability itself
    step = min(1.0, float(size.max()) * 8 * U32)
    close(leaves[1].grad, de, de_size * (2 * u + 1e-5 + 2 * step) + 4 * TINY[dtype], "dtable")
