"""layer_norm and rms_norm on the GPU against their formulas in 64 bits, values and gradients, at every row shape of the
kernels; strides, types, empty and special rows, differences, determinism, streams and captured training steps."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import adambridge_b200 as ab
from adambridge_b200 import native

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
OUT = {torch.float32: E, torch.bfloat16: 2.0 ** -8}     # half a step, relative


def formula(x, w, b, eps, rms, dy=None):
    """y, and with dy also dx, dw, db, in 64 bits; `sizes` are sums of magnitudes that the bounds below refer to."""
    x = x.double()
    mu = torch.zeros_like(x[:, :1]) if rms else x.mean(1, keepdim=True)
    r = 1 / ((x - mu).square().mean(1, keepdim=True) + eps).sqrt()
    h = (x - mu) * r
    ww = torch.ones_like(x[0]) if w is None else w.double()
    bb = torch.zeros_like(x[0]) if b is None else b.double()
    out = {"y": h * ww + bb}
    # what one rounding of mean, deviation and r moves h by, in units of e: n for the sums' lengths
    out["h_size"] = h.abs() + (x.abs() + x.abs().mean(1, keepdim=True)) * r
    if dy is not None:
        dy = dy.double()
        a = dy * ww
        c1 = 0.0 if rms else a.mean(1, keepdim=True)
        c2 = (a * h).mean(1, keepdim=True)
        out["dx"] = r * (a - c1 - h * c2)
        out["dw"], out["db"] = (dy * h).sum(0), dy.sum(0)
        hs = out["h_size"]
        out["dx_size"] = r * (a.abs() + a.abs().mean(1, keepdim=True) + hs * (a.abs() * hs).mean(1, keepdim=True))
        out["dw_size"], out["db_size"] = (dy.abs() * hs).sum(0), dy.abs().sum(0)
    return out


def depth(cols):
    """Roundings on a value's way through a row's sum: one thread's values (at most 32 of them, or cols / 512 in rows
    longer than a CTA's registers, which 512 threads share), then the tree."""
    return max(32, cols / 512) + 12


def check(x, w, b, eps, rms, dy=None, wants=(True, True, True)):
    """Compare with the formula.  Every fp32 operation rounds by at most e = 2^-24 of its result.  A row's mean, variance
    and c1, c2 are sums with at most n = depth(cols) roundings on each value's way, so h is off by at most
    (2 n + 8) e h_size, y by that times |w| plus 2 e (|y| + |b|) and half a step of its type, dx by (4 n + 16) e dx_size
    plus half a step, dw and db by the sums' rows besides: (2 n + 8 + m) e size, m the roundings of the sums over rows."""
    leaves = [t.requires_grad_(k) if t is not None else None for t, k in zip((x, w, b), wants)]
    y = ab.rms_norm(x, w, eps=eps) if rms else ab.layer_norm(x, w, b, eps=eps)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    cols = x.shape[-1]
    flat = lambda t: None if t is None else t.detach().reshape(-1, cols)   # noqa: E731
    want = formula(flat(x), None if w is None else w.detach(), None if b is None else b.detach(), eps, rms, flat(dy))
    n = depth(cols)
    wa = 1.0 if w is None else w.detach().double().abs()
    ba = 0.0 if b is None else b.detach().double().abs()
    off = (flat(y).double() - want["y"]).abs()
    assert bool((off <= (2 * n + 8) * E * want["h_size"] * wa + 2 * E * (want["y"].abs() + ba)
                 + OUT[y.dtype] * want["y"].abs() * (1 + 1e-3) + 1e-37).all()), float(off.max())
    if dy is None:
        return y, None
    asked = [t for t, k in zip(leaves, wants) if t is not None and k]
    grads = dict(zip([name for name, t, k in zip(("dx", "dw", "db"), leaves, wants) if t is not None and k],
                     torch.autograd.grad(y, asked, dy)))
    rows = want["y"].shape[0]
    m = rows / 100 + 64
    for name, got in grads.items():
        k = 4 * n + 16 if name == "dx" else 2 * n + 8 + m
        ref = want[name]
        assert got.dtype == {"dx": x, "dw": w, "db": b}[name].dtype
        off = (got.double().reshape(ref.shape) - ref).abs()
        assert bool((off <= k * E * want[name + "_size"] + OUT[got.dtype] * ref.abs() * (1 + 1e-3) + 1e-37).all()), (
            name, float(off.max()))
    return y, grads


def data(rows, cols, dtype, seed=0, offset=0.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s, dt=dtype, mean=0.0, std=1.0: torch.empty(s, dtype=dt, device="cuda").normal_(mean, std, generator=gen)   # noqa: E731
    return new(rows, cols, mean=offset), new(cols, mean=1.0, std=0.2), new(cols), new(rows, cols)


COLS = [1, 2, 7, 8, 31, 64, 65, 96, 128, 129, 256, 257, 264, 512, 1000, 1024, 1032, 2048, 2049, 4096, 4097, 8192, 8200, 11008, 12288,
        20001, 32776]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rms", [False, True])
def test_every_row_shape(cols, dtype, rms):
    for rows in (1, 3, 130) if cols > 300 else (1, 37, 3000):
        x, w, b, dy = data(rows, cols, dtype, cols + rows)
        check(x, w, None if rms else b, 1e-5, rms, dy)


@pytest.mark.parametrize("cols", [2056, 4104, 5120, 6144, 6152, 9001, 10240, 10248, 12296, 15001, 16392, 20480, 20488])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_long_rows(cols, dtype):
    """Enough long rows that each CTA takes several and keeps their sums, which the shapes for long rows need."""
    x, w, b, dy = data(700, cols, dtype, cols)
    check(x, w, b, 1e-5, False, dy)
    check(x.detach(), w.detach(), None, 1e-5, True, dy, (cols % 16 == 0, True, False))


def in_flight(lanes):
    """Rows that every resident CTA together take at once, at most: 2048 threads per SM."""
    return torch.cuda.get_device_properties(0).multi_processor_count * 2048 // lanes


# vectors of a row, and the least number of threads that own one, forward or backward
VECTORS = [(8, 8), (16, 8), (32, 16), (64, 32), (128, 32), (256, 128), (512, 256), (768, 256), (1024, 256), (1536, 512),
           (2048, 512), (2560, 512)]
SINGLES = [(8, 8), (16, 16), (32, 32), (48, 16), (64, 32), (96, 32), (128, 64), (192, 64), (256, 128), (384, 128), (512, 256),
           (768, 256), (1024, 512), (1536, 512), (2048, 512), (2560, 512)]


@pytest.mark.parametrize("vectors, lanes, aligned", [(*s, True) for s in VECTORS] + [(*s, False) for s in SINGLES])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rms", [False, True])
def test_several_rows_per_cta(vectors, lanes, aligned, dtype, rms):
    """Three times the rows that are under way at once and some more: every CTA takes several groups of rows, its ring goes
    around, its sums are carried from group to group, and the last group has a row for some of its threads only."""
    cols = vectors * (16 // dtype.itemsize) - (0 if aligned else 1)
    x, w, b, dy = data(3 * in_flight(lanes) + 13, cols, dtype, cols)
    check(x, w, None if rms else b, 1e-5, rms, dy)


@pytest.mark.parametrize("xt, wt", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("cols", [64, 129, 4096, 4100, 20000])
def test_mixed_types(xt, wt, cols):
    x, w, b, dy = data(70, cols, xt, 1)
    for rms in (False, True):
        check(x.detach(), w.detach().to(wt), None if rms else b.detach().to(wt), 1e-6, rms, dy)


@pytest.mark.parametrize("cols", [100, 1024, 9000])
@pytest.mark.parametrize("wants", [(True, False, False), (False, True, False), (False, False, True), (False, True, True),
                                   (True, False, True)])
def test_gradients_that_are_asked_for(cols, wants):
    x, w, b, dy = data(50, cols, torch.bfloat16, 2)
    check(x, w, b, 1e-5, False, dy, wants)
    if wants[0] or wants[1]:
        check(x.detach(), w.detach(), None, 1e-5, True, dy, wants[:2] + (False,))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_without_weight_or_bias(dtype):
    x, w, b, dy = data(50, 1000, dtype, 3)
    check(x, None, None, 1e-5, False, dy)
    check(x.detach(), None, None, 1e-5, True, dy)
    check(x.detach(), w, None, 1e-5, False, dy)
    check(x.detach(), None, b, 1e-5, False, dy)
    assert torch.equal(ab.layer_norm(x.detach(), w.detach(), b.detach()), ab.layer_norm(x, w, b).detach())   # no grad


@pytest.mark.parametrize("cols", [64, 1000, 4096, 12000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(cols, dtype):
    """Rows in a wider buffer (aligned or not), a transposed batch, permuted and expanded tensors, unaligned starts: what
    a contiguous copy gives, up to the order of a row's sum; and what lies around is left as it was."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.empty(40, cols + 24, dtype=dtype, device="cuda").normal_(generator=gen)
    keep = wide.clone()
    _, w, b, _ = data(1, cols, dtype, 5)
    for at in (0, 8, 3):
        x = wide[:, at:at + cols]
        check(x.detach(), w, b, 1e-5, False, wide[:, 16:16 + cols])
    x = wide[:, :cols].reshape(4, 10, cols)
    check(x.transpose(0, 1), w, b, 1e-5, False, x.transpose(0, 1))
    check(wide[:cols, :40].t()[:, :8] if cols == 64 else wide[::2, :cols], None, None, 1e-5, True,
          torch.ones((), dtype=dtype, device="cuda").expand(40 if cols == 64 else 20, 8 if cols == 64 else cols))
    check(wide[0, :cols].expand(6, cols), w, b, 1e-5, False, wide[:6, :cols])
    odd = torch.empty(cols + 1, dtype=dtype, device="cuda").normal_(generator=gen)[1:]
    check(wide[:, :cols].contiguous(), odd, odd.clone(), 1e-5, False, wide[:, :cols])
    check(wide[0, :cols].detach(), w, b, 1e-5, False, wide[1, :cols])          # one axis
    assert torch.equal(wide, keep)


@pytest.mark.parametrize("which", ["x", "w", "b", "dy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_negated_views(which, dtype):
    """Lazily negated tensors, as the imaginary part of a conjugate is, give what negated copies give."""
    given = dict(zip("x w b dy".split(), data(50, 72, dtype, 4)))
    lazy = dict(given, **{which: torch._neg_view(given[which])})
    given[which] = -given[which]
    results = []
    for t in (given, lazy):
        leaves = [t[k].requires_grad_(True) for k in ("x", "w", "b")]
        y = ab.layer_norm(*leaves)
        results.append([y, *torch.autograd.grad(y, leaves, t["dy"])])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    z = torch.randn(300, 1, dtype=torch.complex64, device="cuda").conj().imag
    assert z.is_neg() and torch.equal(ab.rms_norm(z), ab.rms_norm(z.clone()))


@pytest.mark.parametrize("cols", [1, 3, 9, 33, 61, 121, 129, 250, 505, 1001, 2050, 4097, 5121, 8185, 9001, 17001, 20003])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_between_other_data(dtype, cols):
    """Rows that start and end anywhere in their 16 bytes, alike in all tensors or not, through the C entry points: NaNs
    before the first row, behind the last and between padded ones stay out of the result, and so does the result of them.
    Bounds as in `check`."""
    kernels = native.load()
    lib, e = kernels._lib, 5e-6
    rows = 3000 if cols < 130 else 300 if cols < 6000 else 150     # more than the CTAs that are resident take at once
    n, half = depth(cols), OUT[dtype]
    _, w, b, _ = data(1, cols, dtype, cols)
    for at, pad, out_at in ((0, 0, 0), (1, 0, 1), (3, 8, 3), (5, 0, 2), (0, 3, 0)):
        stride, room = cols + pad, 16
        def place(seed, start, gap):
            gen = torch.Generator(device="cuda").manual_seed(seed)
            buf = torch.full((room + start + rows * (cols + gap) + room,), float("nan"), dtype=dtype, device="cuda")
            view = torch.as_strided(buf, (rows, cols), (cols + gap, 1), room + start)
            view.normal_(0.5, 1.0, generator=gen)
            return buf, view
        _, x = place(1, at, pad)
        _, dy = place(2, out_at, 0)
        (ybuf, y), (dxbuf, dx) = place(3, out_at, 0), place(4, out_at, 0)
        stats = torch.empty(2, rows, device="cuda")
        spec = native.Norm(x=x.data_ptr(), w=w.data_ptr(), b=b.data_ptr(), rows=rows, cols=cols, x_stride=stride,
                           dtype=native.dtype_code_of(dtype), w_dtype=native.dtype_code_of(dtype), rms=0, eps=e)
        stream = torch.cuda.current_stream().cuda_stream
        p = ctypes.byref(spec)
        assert lib.abx_norm_forward(stream, p, y.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr()) == 0
        size = lib.abx_norm_backward_workspace_bytes(p)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        dw, db = torch.empty_like(w), torch.empty_like(b)
        assert lib.abx_norm_backward(stream, p, dy.data_ptr(), cols, stats[0].data_ptr(), stats[1].data_ptr(), dx.data_ptr(),
                                     dw.data_ptr(), db.data_ptr(), ws.data_ptr(), size) == 0
        want = formula(x, w, b, spec.eps, False, dy)
        wa, m = w.double().abs(), rows / 100 + 64
        bounds = {"y": (y, (2 * n + 8) * E * want["h_size"] * wa + 2 * E * (want["y"].abs() + b.double().abs())),
                  "dx": (dx, (4 * n + 16) * E * want["dx_size"]), "dw": (dw, (2 * n + 8 + m) * E * want["dw_size"]),
                  "db": (db, (2 * n + 8 + m) * E * want["db_size"])}
        for name, (got, bound) in bounds.items():
            off = (got.double() - want[name]).abs()
            assert bool((off <= bound + half * want[name].abs() * (1 + 1e-3) + 1e-37).all()), (name, at, pad, float(off.max()))
        for buf, view in ((ybuf, y), (dxbuf, dx)):
            view.fill_(float("nan"))
            assert bool(buf.isnan().all())


def test_no_rows():
    w, b = (torch.randn(64, device="cuda", requires_grad=True) for _ in range(2))
    x = torch.zeros(0, 5, 64, device="cuda", requires_grad=True)
    y = ab.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert y.shape == dx.shape == (0, 5, 64)
    assert float(dw.abs().max()) == float(db.abs().max()) == 0.0


@pytest.mark.parametrize("cols", [64, 1000, 4096, 20000])
def test_special_rows(cols):
    """A row with a NaN or an infinity is NaN where the formula's is and leaves its neighbours alone; a constant row gives the
    bias; large offsets do not cancel the variance away."""
    x, w, b, dy = data(6, cols, torch.float32, 6)
    plain = ab.layer_norm(x, w, b)
    x[1, 3], x[3, 5], x[4] = float("nan"), float("inf"), 7.0
    y = ab.layer_norm(x, w, b)
    assert bool(y[1].isnan().all()) and bool(y[3].isnan().all())
    assert torch.equal(y[[0, 2, 5]], plain[[0, 2, 5]])
    # the mean of equal values is off by n roundings at most, and h = (x - mean) / sqrt(var + eps) by that over sqrt(eps)
    assert bool(((y[4] - b).abs() <= depth(cols) * E * 7.0 / math.sqrt(1e-5) * w.abs() + 2 * E * b.abs()).all())
    assert bool(ab.rms_norm(x, w)[1].isnan().all())
    far, _, _, _ = data(6, cols, torch.float32, 7, offset=1000.0)
    check(far, w, b, 1e-5, False, dy)


@pytest.mark.parametrize("cols", [1, 4, 5, 20, 40, 65, 300, 1000, 1023, 4100, 4099, 9001, 12004, 20001, 20004])
def test_constant_rows_of_large_values(cols):
    """Every value 2^112, whose sum and mean are exact: h is 0, and dx = r (a - mean a), although -mean r, which h would be
    beyond the row's end, overflows.  Each of a, its mean (n roundings) and dx rounds: (n + 8) e r (|a| + mean |a|)."""
    if float(torch.tensor(float(cols)) * (1.0 / torch.tensor(float(cols)))) != 1.0:
        pytest.skip("the reciprocal's rounding moves the mean")
    _, w, b, dy = data(40, cols, torch.float32, 13)
    x = torch.full((40, cols), 2.0 ** 112, device="cuda", requires_grad=True)
    w.requires_grad_(True)
    b.requires_grad_(True)
    eps = 1e-12
    y = ab.layer_norm(x, w, b, eps=eps)
    assert torch.equal(y, b.expand(40, cols))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    a = dy.double() * w.detach().double()
    r = 1 / math.sqrt(float(torch.tensor(eps)))
    want = r * (a - a.mean(1, keepdim=True))
    size = r * (a.abs() + a.abs().mean(1, keepdim=True))
    assert bool(((dx.double() - want).abs() <= (depth(cols) + 8) * E * size).all())
    assert float(dw.abs().max()) == 0.0
    assert bool(((db.double() - dy.double().sum(0)).abs() <= 80 * E * dy.double().abs().sum(0)).all())


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("cols", [5, 40, 300])
def test_gradients_against_differences(rms, cols):
    """The analytic gradient of sum(y * c) against central differences of the formula in 64 bits, step 1e-4: their error is
    about 1e-8 of the third derivative's size, the kernel's a few hundred e; 1e-4 of the gradient's scale covers both."""
    x, w, b, c = data(7, cols, torch.float32, 8)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = ab.rms_norm(x, w) if rms else ab.layer_norm(x, w, b)
    dx, dw = torch.autograd.grad((y * c).sum(), (x, w))
    f = lambda xx, ww: float((formula(xx, ww, None if rms else b, 1e-5, rms)["y"] * c.double()).sum())   # noqa: E731
    gen = torch.Generator(device="cuda").manual_seed(9)
    for _ in range(5):
        vx = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)
        vw = torch.randn(w.shape, generator=gen, device="cuda", dtype=torch.float64)
        s = 1e-4
        xd, wd = x.detach().double(), w.detach().double()
        slope = (f(xd + s * vx, wd + s * vw) - f(xd - s * vx, wd - s * vw)) / (2 * s)
        got = float((dx.double() * vx).sum() + (dw.double() * vw).sum())
        scale = float((dx.double() * vx).abs().sum() + (dw.double() * vw).abs().sum())
        assert abs(got - slope) <= 1e-4 * scale


@pytest.mark.parametrize("rows, cols", [(5000, 128), (3000, 4096), (300, 20000)])
def test_the_same_bits_again(rows, cols):
    x, w, b, dy = data(rows, cols, torch.bfloat16, 10)
    first = check(x, w, b, 1e-5, False, dy)[1]
    for _ in range(3):
        y = ab.layer_norm(x, w, b)
        again = torch.autograd.grad(y, (x, w, b), dy)
        assert all(torch.equal(a, f) for a, f in zip(again, first.values()))


def test_another_stream_and_in_place_changes():
    x, w, b, dy = data(2000, 4096, torch.bfloat16, 11)
    want = ab.layer_norm(x, w, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ab.layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want, got)
    w.requires_grad_(True)
    y = ab.layer_norm(x, w, b)
    x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_long_rows_of_different_lengths_on_two_threads():
    """The long kernels ask for shared memory by the row's length; calls at the same time do not take each other's away."""
    import threading
    lib = native.load()._lib
    streams = [torch.cuda.Stream() for _ in range(2)]
    codes: list[set] = [set(), set()]
    held = []
    for cols in (27000, 54000):                 # 108 and 216 KB of fp32
        held.append((torch.ones(1, cols, device="cuda"), torch.empty(1, cols, device="cuda")))
    torch.cuda.synchronize()

    def work(k):
        x, y = held[k]
        spec = native.Norm(x=x.data_ptr(), rows=1, cols=x.shape[1], x_stride=x.shape[1], dtype=native.DT_F32,
                           w_dtype=native.DT_F32, rms=1, eps=1e-5)
        for _ in range(5000):
            codes[k].add(lib.abx_norm_forward(streams[k].cuda_stream, ctypes.byref(spec), y.data_ptr(), None, None))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [{0}, {0}]
    for _, y in held:
        assert bool(((y - 1 / math.sqrt(1 + 1e-5)).abs() <= 4 * E).all())


def test_past_32_bits():
    """More than 2^32 values: the last rows equal the same rows alone."""
    if torch.cuda.get_device_properties(0).total_memory < 80 << 30:
        pytest.skip("needs 80 GB")
    cols = 4096
    rows = 2 ** 32 // cols + 100
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    tail, w, b, dy = data(100, cols, torch.bfloat16, 12)
    x[-100:] = tail
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = ab.layer_norm(x, w, b)
    assert torch.equal(y.detach()[-100:], ab.layer_norm(tail, w.detach(), b))
    d = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    d[-100:] = dy
    dx, dw = torch.autograd.grad(y, (x, w), d)
    short = tail.clone().requires_grad_(True)
    sx, sw = torch.autograd.grad(ab.layer_norm(short, w, b), (short, w), dy)
    assert torch.equal(dx[-100:], sx)
    torch.testing.assert_close(dw, sw, rtol=2 * 2.0 ** -8, atol=1e-2)    # another order of the sum over rows
    del x, y, d, dx
    torch.cuda.empty_cache()


def test_refusals():
    x, w, b, _ = data(4, 64, torch.float32)
    for bad, kind, message in ((dict(weight=w[:32]), ValueError, "shape"), (dict(bias=b[:, None]), ValueError, "shape"),
                               (dict(weight=w.half()), TypeError, "float32 or bfloat16"),
                               (dict(weight=w, bias=b.bfloat16()), TypeError, "one dtype"),
                               (dict(weight=w.cpu()), ValueError, "is on"), (dict(eps=-1.0), ValueError, "epsilon"),
                               (dict(eps=float("nan")), ValueError, "epsilon")):
        with pytest.raises(kind, match=message):
            ab.layer_norm(x, **bad)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ab.rms_norm(x.half(), w)
    x.requires_grad_(True)
    g, = torch.autograd.grad(ab.rms_norm(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(which, grad):
    """A tangent that went nowhere would read as a derivative of 0."""
    import torch.autograd.forward_ad as forward_ad
    args = [t.detach() for t in data(4, 64, torch.float32)[:3]]
    args[0].requires_grad_(grad)
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ab.layer_norm(*args)
        if which < 2:
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                ab.rms_norm(*args[:2])
    x, w, _, dy = data(4, 64, torch.float32)
    y = ab.rms_norm(x.requires_grad_(True), w)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        torch.autograd.grad(y, x, forward_ad.make_dual(dy, torch.ones_like(dy)))


def test_traces_and_transforms_are_refused():
    """They would record a result that nothing computes, or cannot reach the values."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, b, _ = data(4, 64, torch.float32)
    for fn in (lambda t: ab.layer_norm(t, w, b), lambda t: ab.rms_norm(t, w)):
        with pytest.raises(Exception, match="trace does not see"):
            torch.jit.trace(fn, (x,))
        with pytest.raises(NotImplementedError, match="trace does not see"):
            make_fx(fn)(x)
        with pytest.raises(NotImplementedError, match="trace does not see"), FakeTensorMode(allow_non_fake_inputs=True) as mode:
            fn(mode.from_tensor(x))
        for transformed in (torch.func.vmap(fn), torch.func.grad(lambda t: fn(t).sum()),
                            lambda t: torch.func.jvp(fn, (t,), (torch.ones_like(t),))):
            with pytest.raises(RuntimeError):
                transformed(x)


# --------------------------------------------------------------------------- a training step of these operators

class Net(torch.nn.Module):
    """Two residual blocks of a norm and two matrices, as a decoder's MLP has them."""

    def __init__(self, width, dtype, seed):
        super().__init__()
        gen = torch.Generator(device="cuda").manual_seed(seed)
        new = lambda *s, std: torch.nn.Parameter(torch.empty(s, device="cuda").normal_(0, std, generator=gen).to(dtype))   # noqa: E731
        one = lambda: torch.nn.Parameter(torch.ones(width, device="cuda", dtype=dtype))   # noqa: E731
        self.up = torch.nn.ParameterList([new(2 * width, width, std=width ** -0.5) for _ in range(2)])
        self.down = torch.nn.ParameterList([new(width, 2 * width, std=(2 * width) ** -0.5) for _ in range(2)])
        self.norm = torch.nn.ParameterList([one() for _ in range(3)])
        self.bias = torch.nn.Parameter(torch.zeros(width, device="cuda", dtype=dtype))

    def forward(self, x):
        for up, down, w in zip(self.up, self.down, self.norm):
            h = torch.nn.functional.silu(ab.rms_norm(x, w) @ up.t())
            x = x + h @ down.t()
        return ab.layer_norm(x, self.norm[2], self.bias)


@pytest.mark.parametrize("precision, width", [("fp32", 256), ("int8", 256), ("int8", 4096)])
def test_a_captured_training_step_equals_eager_ones(precision, width):
    """Norms, their gradients, the clip and the update in one graph: five replays on new batches equal five eager steps."""
    def build():
        net = Net(width, torch.bfloat16, 1)
        return net, ab.GraphAdamW(net.parameters(), lr=1e-2, precision=precision, seed=3)

    def step(net, opt, x, target):
        opt.zero_grad(set_to_none=True)
        loss = (net(x) - target).float().square().mean()
        loss.backward()
        opt.clip_grad_norm_(0.05)
        opt.step()
        return loss

    gen = torch.Generator(device="cuda").manual_seed(2)
    batches = [[torch.empty(96, width, dtype=torch.bfloat16, device="cuda").normal_(generator=gen) for _ in range(2)]
               for _ in range(6)]
    net, opt = build()
    eager = [float(step(net, opt, *batch)) for batch in batches]

    other, graphed = build()
    x, target = batches[0][0].clone(), batches[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        losses = [float(step(other, graphed, x, target))]       # the warm-up is the first step
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(other, graphed, x, target)
    for batch in batches[1:]:
        x.copy_(batch[0])
        target.copy_(batch[1])
        graph.replay()
        losses.append(float(loss))
    assert losses == eager
    assert graphed.arenas[0].steps.tolist() == [6] * len(list(other.parameters()))
    for a, b in zip(net.parameters(), other.parameters()):
        assert torch.equal(a, b)
