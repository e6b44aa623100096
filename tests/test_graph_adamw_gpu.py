"""GraphAdamW on the GPU, against the formulas in 64 bits (bounds derived from the roundings) and against an fp32
restatement of them on the CPU (bit for bit): every state and weight format, sizes around the block, vector and tile,
unaligned and strided tensors, skipped steps, capture and replay, checkpoints."""

from __future__ import annotations

import math

import pytest
import torch

import adambridge_b200 as ab

pytestmark = pytest.mark.gpu

BLOCK = 256
E = 2.0 ** -24            # half a step of fp32, relative
HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
SIZES = [1, 7, 8, 255, 256, 257, 2047, 2048, 2049, 5000, 0, 70001]


def make(sizes, dtype, seed=0, scale=1e-3, **kw):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    params = []
    for n in sizes:
        p = torch.nn.Parameter(torch.empty(n, dtype=dtype, device="cuda").normal_(0, 0.02, generator=gen))
        p.grad = torch.empty(n, dtype=dtype, device="cuda").normal_(0, scale, generator=gen)
        params.append(p)
    return params, ab.GraphAdamW(params, **{**HYPER, **kw})


def new_gradients(params, seed, scale=1e-3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for p in params:
        p.grad.copy_(torch.empty_like(p.grad).normal_(0, scale, generator=gen))


def hash32(x):
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def state_of(opt, arena, i):
    """(p, m, v, m scale, v scale) of parameter i on the CPU, fp32 values; scales per value."""
    at, n = arena.offsets[i], arena.numels[i]
    p = arena.master_of(i).cpu().clone()
    m, v = arena.exp_avg()[at:at + n].cpu().clone(), arena.exp_avg_sq()[at:at + n].cpu().clone()
    if opt.precision == "fp32":
        return p, m, v, None, None
    blocks = torch.arange(n) // BLOCK + at // BLOCK
    return p, m, v, arena.m_scale.cpu()[blocks], arena.v_scale.cpu()[blocks]


def restated(p, m, v, g, step, index, scale, opt):
    """The step on the CPU, fp32, each operation rounded once: (p, m, v) and, for 8-bit states, decoded new moments."""
    lr, (b1, b2), eps, wd = HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"]
    g = g.float()
    if scale is not None:
        g = g * torch.tensor(scale)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * (1 - b2) * g
    r = torch.sqrt(v.double()).float()    # rounded correctly, which the CPU's vector sqrt is not always
    p = p * (1 - lr * wd) - m / (r * (1 / math.sqrt(1 - b2 ** step)) + eps) * (lr / (1 - b1 ** step))
    if opt.precision == "fp32":
        return p, m, v
    n = p.numel()
    pad = lambda x: torch.cat([x, torch.zeros(-n % BLOCK)]).view(-1, BLOCK)   # noqa: E731
    m, r = pad(m), pad(r)
    words = hash32(torch.arange(m.numel()) ^ hash32(hash32(torch.tensor(hash32(opt.seed) ^ index)) ^ step)).view(-1, BLOCK)
    um, uv = (words & 0xFFFF).float() / 65536, (words >> 16).float() / 65536
    below = torch.nextafter(torch.tensor([127.0, 255.0]), torch.zeros(2))
    tm, tr = m.abs().amax(1, keepdim=True), r.amax(1, keepdim=True)
    x = m * torch.where(tm > 2.0 ** -100, below[0] / tm, 0.0)
    qm = torch.floor(x + um) if opt.stochastic else torch.round(x)
    x = r * torch.where(tr > 2.0 ** -100, below[1] / tr, 0.0)
    if opt.stochastic:
        q = torch.floor(x)
        q = q + ((x - q) * (x + q) > uv * (q + q + 1)).float()
    else:
        q = torch.round(x)
    q = torch.where(r > 0, q.clamp(min=1), q)
    sm = torch.where(tm > 2.0 ** -100, tm * torch.tensor(1 / 127), 0.0)
    sv = torch.where(tr > 2.0 ** -100, tr * torch.tensor(1 / 255), 0.0)
    return p, (qm * sm).view(-1)[:n], (q * sv).square().view(-1)[:n]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("precision, stochastic", [("fp32", True), ("int8", True), ("int8", False)])
@pytest.mark.parametrize("scale", [None, 0.37])
def test_bits_equal_the_fp32_restatement(dtype, precision, stochastic, scale):
    params, opt = make(SIZES, dtype, 3, precision=precision, stochastic_rounding=stochastic)
    opt.seed = 5
    arena = opt.prepare().arenas[0]
    factor = None if scale is None else torch.full((1,), scale, device="cuda")
    for step in (1, 2, 3):
        new_gradients(params, 10 + step)
        want = [restated(*state_of(opt, arena, i)[:3], p.grad.cpu(), step, i, scale, opt) for i, p in enumerate(params)]
        opt.step(grad_scale=factor)
        for i, (p, (wp, wm, wv)) in enumerate(zip(params, want)):
            gp, gm, gv, _, _ = state_of(opt, arena, i)
            assert torch.equal(gm, wm) and torch.equal(gv, wv), (i, step)
            assert torch.equal(gp, wp), (i, step)
            assert torch.equal(p.detach().cpu(), wp.to(dtype)), (i, step)
    assert arena.steps.tolist() == [3 if n else 0 for n in SIZES]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("precision, stochastic", [("fp32", True), ("int8", True), ("int8", False)])
@pytest.mark.parametrize("spread", [1e-3, 1.0])
def test_against_64_bits(dtype, precision, stochastic, spread):
    """One step from a state of several steps.  With e = 2^-24: m is off by at most 4 e S, S = |b1 m| + |(1-b1) g| (the
    coefficient's, the product's, the scaled gradient's and the sum's rounding); v, a sum of positive terms, by 6 e v; the
    denominator by (3 + 3) e of itself; so the update by a / d (4 e S + 8 e |m|), and p by 2 e |p| + e |p'| more."""
    params, opt = make([3000, 257], dtype, 4, scale=spread, precision=precision, stochastic_rounding=stochastic)
    arena = opt.prepare().arenas[0]
    for step in range(1, 5):
        new_gradients(params, 20 + step, spread)
        if step < 4:
            opt.step()
    before = [state_of(opt, arena, i) for i in range(2)]
    opt.step(grad_scale=torch.full((1,), 0.5, device="cuda"))
    (b1, b2), lr, t = HYPER["betas"], HYPER["lr"], 4
    for i, param in enumerate(params):
        p, m, v = (x.double() for x in before[i][:3])
        g = param.grad.cpu().double() * 0.5
        m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        d = (v1 / (1 - b2 ** t)).sqrt() + HYPER["eps"]
        a = lr / (1 - b1 ** t)
        p1 = p * (1 - lr * HYPER["weight_decay"]) - a * m1 / d
        s = (b1 * m).abs() + ((1 - b1) * g).abs()
        gp, gm, gv, sm, sv = state_of(opt, arena, i)
        slack = E * (2 * p.abs() + p1.abs() + a / d * (4 * s + 8 * m1.abs()))
        assert bool(((gp.double() - p1).abs() <= slack).all())
        off_m, off_r = 4 * E * s, 4 * E * v1.sqrt()
        if precision == "int8":
            # a code: half of one, or one, by the rounding; x and the scale have 3 roundings of |x| <= 255
            off_m = off_m + sm.double() * ((1.0 if stochastic else 0.5) + 127 * 4 * E)
            off_r = off_r + sv.double() * ((1.0 if stochastic else 0.5) + 255 * 4 * E)
            # below one code a positive root is stored as one
            off_r = torch.where(v1.sqrt() < sv.double(), sv.double() * (1 + 4 * E), off_r)
            assert bool((gv[v1 > 0] > 0).all())
        assert bool(((gm.double() - m1).abs() <= off_m).all())
        assert bool(((gv.double().sqrt() - v1.sqrt()).abs() <= off_r + 2 * E * v1.sqrt()).all())


def plain_step(m, v, eps):
    """One fp32 step with zero gradients from the moments m, v.  Decays of 1/2 halve them, after 200 steps the bias
    corrections are 1, and the learning rate is 1: a weight of 0 becomes -(m' / (sqrt(v') + eps)).  Returns that and what
    64 bits say, rounded once at each operation (a root or quotient of two floats in 53 bits rounds to the right one)."""
    p = torch.nn.Parameter(torch.zeros_like(m))
    p.grad = torch.zeros_like(m)
    opt = ab.GraphAdamW([p], lr=1.0, betas=(0.5, 0.5), eps=eps, weight_decay=0.0, precision="fp32").prepare()
    a, n = opt.arenas[0], m.numel()
    a.m[:n].copy_(m)
    a.v[:n].copy_(v)
    a.steps.fill_(200)
    opt.step()
    m, v = a.m[:n], a.v[:n]
    d = v.double().sqrt().float() + torch.tensor(eps, dtype=torch.float32, device="cuda")
    return p.detach(), -(m.double() / d.double()).float()


def test_roots_of_every_second_moment():
    """Every float of [2^-104, 2^50), which is what the fast root takes and some of what it does not on either side."""
    start, stop, at_once = 23 << 23, 177 << 23, 1 << 26
    gen = torch.Generator(device="cuda").manual_seed(1)
    for at in range(start, stop, at_once):
        bits = torch.arange(at, min(at + at_once, stop), dtype=torch.int32, device="cuda")
        v = bits.view(torch.float32) * 2
        got, want = plain_step(torch.empty_like(v).uniform_(0.5, 2.0, generator=gen), v, 0.0)
        assert torch.equal(got, want), at


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-8, 1.0, 2.0 ** 24, 2.0 ** 40, 2.0 ** 100])
@pytest.mark.parametrize("low, high", [(-149, -100), (-149, 60), (-101, 0)])
def test_quotients_of_first_moments_of_any_size(low, high, eps):
    """First moments that decayed to 2^-149 beside second moments of any size, zeros among both: the quotient is the IEEE
    one, also where it or the remainder that corrects it leaves the range of normal numbers."""
    n = (1 << 22) + 1000
    gen = torch.Generator(device="cuda").manual_seed(2)
    def spread(a, b):
        e = torch.empty(n, device="cuda", dtype=torch.float64).uniform_(a, b, generator=gen)
        return torch.exp2(e).float()
    m, v = spread(low, high), spread(-140, 120)
    m *= torch.where(torch.rand(n, device="cuda", generator=gen) < 0.5, -1.0, 1.0)
    # blocks of moments of ordinary size too: zeros and small ones among them decide which way a block goes
    v[: n // 2] = spread(-60, 20)[: n // 2]
    m[::1001] = 0.0
    if eps > 0:
        v[::997] = 0.0
    got, want = plain_step(m, v, eps)
    assert torch.equal(got, want), int((got != want).sum())


def test_decayed_moments_of_zero_weights():
    """Rows of an embedding that get no more gradients: bit for bit, as the moments decay below 2^-100."""
    params, opt = make([70001], torch.float32, 3, precision="fp32")
    params[0].data.zero_()
    opt.step()
    arena = opt.arenas[0]
    arena.m.mul_(2.0 ** -85)
    params[0].data.zero_()
    params[0].grad.zero_()
    for step in range(2, 60):
        params[0].data.zero_()
        want = restated(*state_of(opt, arena, 0)[:3], params[0].grad.cpu(), step, 0, None, opt)
        opt.step()
        assert all(torch.equal(a, b) for a, b in zip(state_of(opt, arena, 0)[:3], want)), step


def test_stochastic_rounding_is_unbiased():
    """One value of m and of v repeated n times beside a large one per block: the mean of what is stored is within six
    standard errors of the value; a code's spread is at most half a step (m), half of (q+1)^2 - q^2 steps (v)."""
    n = 256 * 2000
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    g = torch.full((n,), 0.1234, device="cuda")
    g[::256] = 1.0
    p.grad = g
    opt = ab.GraphAdamW([p], **HYPER, precision="int8")
    opt.step()
    arena = opt.arenas[0]
    small = torch.arange(n, device="cuda") % 256 != 0
    for got, value, step in ((arena.exp_avg(), 0.1 * 0.1234, 0.1 / 127),
                             (arena.exp_avg_sq(), 1e-3 * 0.1234 ** 2, (2 * 0.1234 * 255 + 2) * 1e-3 / 255 ** 2)):
        got = got[small].double()
        assert got.unique().numel() == 2
        assert abs(float(got.mean()) - value) < 6 * step / 2 / math.sqrt(got.numel()) + 1e-5 * value


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("precision, stochastic", [("fp32", True), ("int8", True), ("int8", False)])
@pytest.mark.parametrize("max_ctas", [1, 3])
def test_few_ctas_give_the_same_bits(dtype, precision, stochastic, max_ctas):
    """One CTA that goes through every tile of every tensor, its ring of blocks many times around, writes what many do:
    weights, moments, scales, masters."""
    sizes = [70001, 1024, 5, 40960, 1023, 9 * 1024 + 8]
    kw = dict(precision=precision, stochastic_rounding=stochastic)
    (one, few), (two, many) = make(sizes, dtype, 3, max_ctas=max_ctas, **kw), make(sizes, dtype, 3, **kw)
    for step in range(3):
        for params, opt in ((one, few), (two, many)):
            new_gradients(params, 30 + step)
            opt.step(grad_scale=torch.full((1,), 0.7, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(snapshot(one, few), snapshot(two, many)))


@pytest.mark.parametrize("codes, stored", [(0.04, 1.0), (0.5, 1.0), (0.999, 1.0), (1.25, None), (7 + 2.0 ** -10, None)])
def test_stochastic_rounding_near_whole_codes(codes, stored):
    """What is stored for a root of so many codes.  Below one code it is always one: a positive v never becomes 0.  Above, v's
    mean is v, within six standard errors and 2^-16 of the gap between the neighbours, as the draw has 16 bits."""
    n = 256 * 4000
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    g = torch.full((n,), codes / 255, device="cuda")
    g[::256] = 1.0
    p.grad = g
    opt = ab.GraphAdamW([p], **HYPER, precision="int8")
    opt.step()
    arena = opt.arenas[0]
    small = torch.arange(n, device="cuda") % 256 != 0
    q = arena.v[:n][small].double()
    if stored is not None:
        assert bool((q == stored).all())
    else:
        low = math.floor(codes)
        gap = 2 * low + 1
        chance = (codes ** 2 - low ** 2) / gap
        spread = math.sqrt(chance * (1 - chance) / q.numel())
        # codes is off by the roundings of g, v, its root and the scale: 6 of 2^-24, relative, twice that in v
        assert abs(float((q * q).mean()) - codes ** 2) <= gap * (6 * spread + 2.0 ** -16) + 12 * E * codes ** 2


@pytest.mark.parametrize("codes", [0.25, 3 + 2.0 ** -10, 100 + 2.0 ** -6])
def test_stochastic_rounding_of_m_near_whole_codes(codes):
    """m's mean is m within six standard errors and 2^-16 of a code."""
    n = 256 * 4000
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    g = torch.full((n,), codes / 127, device="cuda")
    g[::256] = 1.0
    p.grad = g
    opt = ab.GraphAdamW([p], **HYPER, precision="int8")
    opt.step()
    small = torch.arange(n, device="cuda") % 256 != 0
    q = opt.arenas[0].m[:n][small].double()
    part = codes - math.floor(codes)
    spread = math.sqrt(part * (1 - part) / q.numel())
    # roundings: g, m, the factor, the product, and of the sum with the draw half of 2^-17 (its step below 128 is 2^-17)
    assert abs(float(q.mean()) - codes) <= 6 * spread + 2.0 ** -16 + 2.0 ** -18 + 8 * E * codes


def test_padding_stays_zero():
    """With eps 0 the padding's update would be 0 / 0."""
    params, opt = make([3, 300], torch.bfloat16, 1, eps=0.0, precision="int8")
    for _ in range(2):
        opt.step()
    a = opt.arenas[0]
    for flat in (a.master, a.exp_avg(), a.exp_avg_sq()):
        for at, n in zip(a.offsets, a.numels):
            rest = flat[at + n:at + -(-n // BLOCK) * BLOCK]
            assert float(rest.abs().max()) == 0.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("precision", ["fp32", "int8"])
@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan")])
def test_padding_stays_zero_whatever_the_gradient_scale(precision, dtype, scale):
    """8-bit moments of such a block are NaN as a whole; the masters' padding and fp32 moments' stays 0."""
    params, opt = make([3, 300], dtype, 1, precision=precision)
    opt.step()
    opt.step(grad_scale=torch.full((1,), scale, device="cuda"))
    a = opt.arenas[0]
    planes = [(a.m, a.offsets), (a.v, a.offsets)] if precision == "fp32" else []
    planes += [(a.master, a.master_offsets)] if a.master is not None else []
    for flat, offsets in planes:
        for at, n in zip(offsets, a.numels):
            rest = flat[at + n:at + -(-n // BLOCK) * BLOCK]
            assert float(rest.abs().max()) == 0.0
    assert bool(a.exp_avg_sq()[:3].isnan().all() or a.exp_avg_sq()[:3].isinf().all())


def test_small_second_moments_never_become_zero_and_updates_stay_bounded():
    p = torch.nn.Parameter(torch.zeros(512, device="cuda"))
    p.grad = torch.full((512,), 1e-6, device="cuda")
    p.grad[0] = 100.0
    opt = ab.GraphAdamW([p], lr=1.0, weight_decay=0.0, eps=0.0, precision="int8", stochastic_rounding=False)
    for _ in range(5):
        before = p.detach().clone()
        opt.step()
        assert float((p.detach() - before).abs().max()) <= 10.0      # Adam's bound (1-b1)/sqrt(1-b2), with room
        assert bool((opt.arenas[0].exp_avg_sq() > 0).all())


@pytest.mark.parametrize("precision", ["fp32", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_unaligned_strided_and_neighbours(precision, dtype):
    """Parameters at odd places of a larger buffer and strided gradients give what contiguous aligned copies give, and
    the values around them stay."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    flat = torch.empty(20000, dtype=dtype, device="cuda").normal_(generator=gen)
    spans = [(1, 300), (401, 2049), (3003, 5000), (9001, 1)]
    keep = flat.clone()
    odd, plain = [], []
    for at, n in spans:
        a, b = torch.nn.Parameter(flat[at:at + n]), torch.nn.Parameter(flat[at:at + n].clone())
        wide = torch.empty(n, 3, dtype=dtype, device="cuda").normal_(generator=gen)
        a.grad, b.grad = wide[:, 1], wide[:, 1].contiguous()
        odd.append(a)
        plain.append(b)
    one, two = (ab.GraphAdamW(ps, **HYPER, precision=precision) for ps in (odd, plain))
    for _ in range(2):
        one.step()
        two.step()
    inside = torch.zeros(20000, dtype=torch.bool, device="cuda")
    for (at, n), a, b in zip(spans, odd, plain):
        assert torch.equal(a, b)
        inside[at:at + n] = True
    assert torch.equal(flat[~inside], keep[~inside])
    assert torch.equal(one.arenas[0].exp_avg(), two.arenas[0].exp_avg())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_negated_gradients(dtype):
    """A gradient that is a lazily negated view, as the imaginary part of a conjugate is."""
    (params, opt), (other, plain) = (make([300, 5000], dtype, 3, precision="fp32") for _ in range(2))
    for p, o in zip(params, other):
        p.grad = torch._neg_view(p.grad.clone())
        o.grad.neg_()
    opt.step()
    plain.step()
    assert all(torch.equal(a, b) for a, b in zip(params, other))


def test_missing_gradients_and_mixed_types():
    bf, _ = make([300, 40, 513], torch.bfloat16, 1)
    fp, _ = make([77, 1000], torch.float32, 2)
    params = [bf[0], fp[0], bf[1], fp[1], bf[2]]
    alone = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for a, p in zip(alone, params):
        a.grad = p.grad.clone()
    params[2].grad = alone[2].grad = None
    opt = ab.GraphAdamW(params, **HYPER, precision="int8", stochastic_rounding=False)
    each = [ab.GraphAdamW([a], **HYPER, precision="int8", stochastic_rounding=False) for a in alone]
    keep = params[2].detach().clone()
    for _ in range(3):
        opt.step()
        for o in each:
            o.step()
    for p, a in zip(params, alone):
        assert torch.equal(p, a)
    assert torch.equal(params[2], keep)
    assert opt.arenas[0].steps.tolist() == [3, 3, 0, 3, 3]


@pytest.mark.parametrize("precision", ["fp32", "int8"])
def test_many_tensors(precision):
    """More tensors than one launch takes, of both types in turn; each equals the same tensor alone."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    params = []
    for i in range(1000):
        p = torch.nn.Parameter(torch.empty(1 + (i * 37) % 3000, dtype=(torch.float32, torch.bfloat16)[i % 2],
                                           device="cuda").normal_(generator=gen))
        p.grad = torch.empty_like(p).normal_(generator=gen)
        params.append(p)
    picked = [0, 1, 383, 384, 385, 767, 768, 769, 999]
    alone = [torch.nn.Parameter(params[i].detach().clone()) for i in picked]
    for a, i in zip(alone, picked):
        a.grad = params[i].grad.clone()
    launched = ab.native.load().launch_count()
    opt = ab.GraphAdamW(params, **HYPER, precision=precision, stochastic_rounding=False)
    opt.step()
    assert ab.native.load().launch_count() - launched == 4      # 500 of each type, 384 per launch
    ab.GraphAdamW(alone, **HYPER, precision=precision, stochastic_rounding=False).step()
    for a, i in zip(alone, picked):
        assert torch.equal(a, params[i]), i
    assert opt.arenas[0].steps.tolist() == [1] * 1000
    assert int(opt.arenas[0].ticket) == 0


def snapshot(params, opt):
    a = opt.arenas[0]
    return [t.clone() for t in (*params, a.m, a.v, a.steps) + ((a.m_scale, a.v_scale) if a.m_scale is not None else ())
            + ((a.master,) if a.master is not None else ())]


@pytest.mark.parametrize("precision", ["fp32", "int8"])
@pytest.mark.parametrize("flag", [1.0, -1.0, float("nan"), float("inf")])
def test_found_inf_changes_nothing(precision, flag):
    params, opt = make([300, 5000], torch.bfloat16, 1, precision=precision)
    opt.step()
    before = snapshot(params, opt)
    opt.step(found_inf=torch.full((1,), flag, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(before, snapshot(params, opt)))
    opt.step(found_inf=torch.zeros(1, device="cuda"))
    assert opt.arenas[0].steps.tolist() == [2, 2]
    assert not torch.equal(before[0], params[0])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_clip_skips_a_step_whose_norm_is_not_finite(bad):
    params, opt = make([300, 5000], torch.bfloat16, 1)
    opt.step()
    before = snapshot(params, opt)
    params[1].grad[17] = bad
    norm = opt.clip_grad_norm_(1.0)
    opt.step()
    assert not math.isfinite(float(norm))
    assert all(torch.equal(a, b) for a, b in zip(before, snapshot(params, opt)))
    params[1].grad[17] = 0.0
    opt.step()                            # the norm of the skipped step is gone
    assert opt.arenas[0].steps.tolist() == [2, 2]


def test_a_gradient_that_is_not_finite_marks_its_block():
    params, opt = make([1024], torch.float32, 1, precision="int8")
    params[0].grad[300] = float("nan")
    params[0].grad[700] = float("inf")
    opt.step()
    for values in (opt.arenas[0].exp_avg(), opt.arenas[0].exp_avg_sq()):
        bad = values.isnan().view(-1, BLOCK)
        assert bad.all(1).tolist() == [False, True, True, False] == bad.any(1).tolist()
    assert params[0].detach().isnan().nonzero().squeeze(1).tolist() == [300, 700]


def test_clip_is_the_coefficient_of_torch():
    params, opt = make([300, 5000], torch.float32, 1, scale=1.0, precision="fp32")
    other, same = make([300, 5000], torch.float32, 1, scale=1.0, precision="fp32")
    total = opt.clip_grad_norm_(0.5)
    want = torch.nn.utils.clip_grad_norm_(other, 0.5)
    torch.testing.assert_close(total, want, rtol=1e-6, atol=0)
    opt.step()
    same.step()
    for a, b in zip(params, other):
        # the first update is a / (1 + eps/|g|)-like: the gradients agree to a few roundings, and so does it
        torch.testing.assert_close(a, b, rtol=4 * E, atol=1e-3 * 16 * E)


@pytest.mark.parametrize("precision", ["fp32", "int8"])
def test_captured_steps_replay(precision):
    """Replays of one captured step equal as many eager steps: counts, rounding, clip, flag and learning rate move on."""
    def build():
        lr = torch.full((1,), 1e-3, dtype=torch.float64, device="cuda")
        params, opt = make([300, 70001, 4096], torch.bfloat16, 6, precision=precision, lr=lr)
        return params, opt, lr, torch.zeros(1, device="cuda")

    def one(opt, flag):
        opt.clip_grad_norm_(1.0)
        opt.step(found_inf=flag)

    eager, graphed = build(), build()
    graphed[1].prepare()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one(graphed[1], graphed[3])
    for k in range(4):
        for params, opt, lr, flag in (eager, graphed):
            new_gradients(params, 50 + k, 1e-2)
            lr.fill_(1e-3 / (k + 1))
            flag.fill_(float(k == 2))
        one(eager[1], eager[3])
        graph.replay()
    for a, b in zip(snapshot(eager[0], eager[1]), snapshot(graphed[0], graphed[1])):
        assert torch.equal(a, b)
    assert graphed[1].arenas[0].steps.tolist() == [3, 3, 3]


def test_clip_of_mixed_gradients_is_captured():
    def build():
        params, _ = make([300, 5000], torch.bfloat16, 6)
        more, _ = make([77, 2000], torch.float32, 7)
        params = [params[0], more[0], params[1], more[1]]
        return params, ab.GraphAdamW(params, **HYPER).prepare()

    eager, graphed = build(), build()
    want = torch.nn.utils.get_total_norm([p.grad.float() for p in eager[0]])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = graphed[1].clip_grad_norm_(1e-3)
        graphed[1].step()
    graph.replay()
    # two norms of four are rounded to bf16
    torch.testing.assert_close(eager[1].clip_grad_norm_(1e-3), want, rtol=2.0 ** -8, atol=0)
    eager[1].step()
    torch.testing.assert_close(total, want, rtol=2.0 ** -8, atol=0)
    for a, b in zip(snapshot(*eager), snapshot(*graphed)):
        assert torch.equal(a, b)


def test_a_clip_and_its_step_are_captured_together():
    params, opt = make([300], torch.bfloat16, 6)
    opt.prepare()
    graph = torch.cuda.CUDAGraph()
    opt.clip_grad_norm_(1.0)
    with pytest.raises(RuntimeError, match="one capture"):
        with torch.cuda.graph(graph):
            opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.clip_grad_norm_(1.0)
    with pytest.raises(RuntimeError, match="one capture"):
        opt.step()
    opt.step()                            # the clip is spent
    assert opt.arenas[0].steps.tolist() == [1]


def test_a_checkpoint_with_a_negative_step_is_refused():
    _, opt = make([300], torch.bfloat16, 6)
    opt.step()
    saved = opt.state_dict()
    saved["state"][0]["step"] = -1
    with pytest.raises(ValueError, match="steps"):
        opt.load_state_dict(saved)
    assert opt.arenas[0].steps.tolist() == [1]


def test_capture_needs_the_state():
    params, opt = make([300], torch.bfloat16, 6)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before a capture"):
        with torch.cuda.graph(graph):
            opt.step()


def test_two_optimizers_on_two_streams():
    """Steps that may overlap (each optimizer has its own ticket) equal steps in turn."""
    sets = [make([70001, 300000], torch.bfloat16, k, precision="int8") for k in (1, 2)]
    alone = [make([70001, 300000], torch.bfloat16, k, precision="int8") for k in (1, 2)]
    for _, opt in sets:
        opt.prepare()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for (_, opt), s in zip(sets, streams):
            with torch.cuda.stream(s):
                opt.step()
    torch.cuda.synchronize()
    for (params, _), (want, opt) in zip(sets, alone):
        for _ in range(5):
            opt.step()
        assert all(torch.equal(a, b) for a, b in zip(params, want))


def test_groups_lr_and_max_ctas():
    params, opt = make([5000, 300], torch.bfloat16, 3, precision="int8")
    more, _ = make([70001], torch.bfloat16, 4)
    opt.add_param_group(dict(params=more, lr=0.0, weight_decay=0.0))
    keep = [p.detach().clone() for p in more]
    opt.step()
    assert all(torch.equal(a, b) for a, b in zip(more, keep))        # lr 0 moves nothing
    assert opt.arenas[1].steps.tolist() == [1] and float(opt.arenas[1].exp_avg().abs().max()) > 0
    one, few = make([70001], torch.bfloat16, 3, max_ctas=1)
    two, all_ = make([70001], torch.bfloat16, 3)
    few.step()
    all_.step()
    assert torch.equal(one[0], two[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_agrees_with_adambridge(dtype):
    """fp32 states: the two differ by fused against separate roundings, a few 2^-24 of the values and of the update."""
    params, opt = make([5000, 300], dtype, 3, precision="fp32")
    other, _ = make([5000, 300], dtype, 3)
    bridge = ab.AdamBridge(other, **HYPER, precision="fp32")
    for k in range(5):
        new_gradients(params, 60 + k)
        new_gradients(other, 60 + k)
        opt.step()
        bridge.step()
    for a, b in zip(opt.master_params(), bridge.master_params()):
        # per step: 3 roundings of |p| <= 0.1 and 16 of an update of at most 1e-3 / 0.1 here
        assert float((a - b.view(-1)).abs().max()) <= 5 * E * (3 * 0.1 + 16 * 1e-2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_between_forward_and_backward_is_noticed(dtype):
    """As torch's optimizers: the backward pass of a graph that saved a weight fails once a step has changed it."""
    params, opt = make([64, 300, 64], dtype, 1)
    params[1].grad = None
    before = [p._version for p in params]
    x = torch.randn(5, 64, device="cuda", dtype=dtype, requires_grad=True)
    kept, other = ab.rms_norm(x, params[0]), ab.rms_norm(x, params[2].detach().clone())
    opt.step()
    assert [p._version > b for p, b in zip(params, before)] == [True, False, True]
    other.sum().backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_clip_on_one_stream_and_its_step_on_another(dtype):
    """The coefficient stays until the step has read it, although the clip's stream goes on and takes free memory."""
    def build():
        params, opt = make([300, 5000], dtype, 6, precision="fp32")
        return params, opt.prepare()

    params, opt = build()
    want, plain = build()
    plain.clip_grad_norm_(1e-3)
    plain.step()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(one):
        opt.clip_grad_norm_(1e-3)
    two.wait_stream(one)
    with torch.cuda.stream(two):
        torch.cuda._sleep(50_000_000)        # some 30 ms
        opt.step()
    with torch.cuda.stream(one):
        taken = [torch.full((k,), 1e6, device="cuda") for k in (1, 2, 4) for _ in range(32)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(snapshot(params, opt), snapshot(want, plain)))
    del taken


def test_a_captured_clip_on_a_forked_stream():
    """Both in one capture, the clip on a stream that the capture forks and joins."""
    (params, opt), (want, plain) = (make([300, 5000], torch.bfloat16, 6) for _ in range(2))
    opt.prepare()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            opt.clip_grad_norm_(1e-3)
        torch.cuda.current_stream().wait_stream(side)
        opt.step()
    for _ in range(3):
        graph.replay()
        plain.clip_grad_norm_(1e-3)
        plain.step()
    assert all(torch.equal(a, b) for a, b in zip(snapshot(params, opt), snapshot(want, plain)))


def test_a_clip_without_gradients_takes_the_last_one_back():
    params, opt = make([300], torch.float32, 6, precision="fp32")
    other, plain = make([300], torch.float32, 6, precision="fp32")
    opt.clip_grad_norm_(1e-3)
    grads = [p.grad for p in params]
    opt.zero_grad(set_to_none=True)
    assert float(opt.clip_grad_norm_(1e-3)) == 0.0
    for p, g in zip(params, grads):
        p.grad = g
    opt.step()
    plain.step()
    assert all(torch.equal(a, b) for a, b in zip(params, other))


# --------------------------------------------------------------------------- checkpoints

@pytest.mark.parametrize("precision", ["fp32", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpoint_resumes_bit_for_bit(precision, dtype):
    params, opt = make([5000, 300, 7], dtype, 3, precision=precision)
    for _ in range(3):
        opt.step()
    saved = {k: v for k, v in torch.load(_saved(opt), weights_only=True).items()}
    again, other = make([5000, 300, 7], dtype, 9, precision=precision)
    for a, p in zip(again, params):
        a.data.copy_(p)
        a.grad.copy_(p.grad)
    other.load_state_dict(saved)
    opt.step()
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(snapshot(params, opt), snapshot(again, other)))


def _saved(opt, **kw):
    import io
    f = io.BytesIO()
    torch.save(opt.state_dict(**kw), f)
    f.seek(0)
    return f


def test_checkpoints_move_to_adambridge_and_back():
    params, opt = make([5000, 300], torch.bfloat16, 3, precision="int8")
    for _ in range(3):
        opt.step()
    other, _ = make([5000, 300], torch.bfloat16, 3)
    bridge = ab.AdamBridge(other, precision="fp32")
    bridge.load_state_dict(opt.state_dict(moments="fp32"))
    arena = opt.arenas[0]
    for i, slot in enumerate(bridge.slots):
        at, n = arena.offsets[i], arena.numels[i]
        assert slot.step == 3
        assert torch.equal(slot.m.to_fp32(), arena.exp_avg()[at:at + n])
        assert torch.equal(slot.v.to_fp32(), arena.exp_avg_sq()[at:at + n])
        assert torch.equal(slot.master.to_fp32(), arena.master_of(i))
    # back, and from FP8 moments: encoded to the nearest codes
    for precision in ("fp32", "fp8"):
        bridge.set_precision(precision)
        _, back = make([5000, 300], torch.bfloat16, 3, precision="int8")
        back.load_state_dict(bridge.state_dict())
        assert back.arenas[0].steps.tolist() == [3, 3]
        for i, slot in enumerate(bridge.slots):
            _, m, v, sm, sv = state_of(back, back.arenas[0], i)
            want_m, want_v = slot.m.to_fp32().cpu(), slot.v.to_fp32().cpu()
            assert bool(((m - want_m).abs() <= sm * (0.5 + 127 * 6 * E)).all())
            off = (v.sqrt() - want_v.sqrt()).abs()
            assert bool((off <= torch.where(want_v.sqrt() < sv, sv, sv * (0.5 + 255 * 6 * E))).all())


def test_torch_adamw_checkpoint_loads():
    params, opt = make([5000, 300], torch.float32, 3, precision="fp32")
    other, _ = make([5000, 300], torch.float32, 3)
    ref = torch.optim.AdamW(other, lr=1e-3)
    ref.step()
    opt.load_state_dict(ref.state_dict())
    for i, p in enumerate(other):
        assert torch.equal(state_of(opt, opt.arenas[0], i)[1], ref.state[p]["exp_avg"].cpu())
    assert opt.arenas[0].steps.tolist() == [1, 1]


def test_load_keeps_the_learning_rate_tensor_that_a_graph_reads():
    lr = torch.full((1,), 1e-3, device="cuda")
    params, opt = make([300], torch.bfloat16, 3, lr=lr)
    opt.step()
    saved = opt.state_dict()
    saved["param_groups"][0]["lr"] = 5e-4
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] is lr and float(lr) == pytest.approx(5e-4)


@pytest.mark.parametrize("change, message", [
    (lambda e: e.pop("exp_avg_sq"), "exp_avg_sq"), (lambda e: e["exp_avg"].update(block=128), "blocks"),
    (lambda e: e["exp_avg"].update(role="v"), "role"), (lambda e: e["exp_avg"].update(q=e["exp_avg"]["q"][:256]), "elements"),
    (lambda e: e["exp_avg_sq"].update(q=e["exp_avg_sq"]["q"].view(torch.int8)), "uint8"),
    (lambda e: e.update(master=torch.zeros(3)), "elements")])
def test_bad_checkpoints_change_nothing(change, message):
    params, opt = make([5000], torch.bfloat16, 3, precision="int8")
    opt.step()
    saved = torch.load(_saved(opt), weights_only=True)
    change(saved["state"][0])
    opt.step()
    before = snapshot(params, opt)
    with pytest.raises(ValueError, match=message):
        opt.load_state_dict(saved)
    assert all(torch.equal(a, b) for a, b in zip(before, snapshot(params, opt)))


@pytest.mark.parametrize("precision", ["fp32", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_checkpoint_replaces_the_whole_state(precision, dtype):
    """Saved before the first step and loaded after some: what a new optimizer on the same weights has, in the same
    buffers, which captured graphs address."""
    params, opt = make([5000, 300, 7], dtype, 3, precision=precision)
    weights = [p.detach().clone() for p in params]
    saved = torch.load(_saved(opt), weights_only=True)
    for _ in range(3):
        opt.step()
    buffers = lambda: [t.data_ptr() for t in (opt.arenas[0].m, opt.arenas[0].v, opt.arenas[0].steps)]   # noqa: E731
    where = buffers()
    for p, w in zip(params, weights):
        p.data.copy_(w)
    opt.load_state_dict(saved)
    fresh, new = make([5000, 300, 7], dtype, 3, precision=precision)
    new.prepare()
    assert all(torch.equal(a, b) for a, b in zip(snapshot(params, opt), snapshot(fresh, new)))
    assert buffers() == where
    for o in (opt, new):
        o.step()
    assert all(torch.equal(a, b) for a, b in zip(snapshot(params, opt), snapshot(fresh, new)))


@pytest.mark.parametrize("precision", ["fp32", "int8"])
def test_a_parameter_that_a_checkpoint_lacks_starts_over(precision):
    params, opt = make([5000, 300, 7], torch.bfloat16, 3, precision=precision)
    lacking, partial = make([5000, 300, 7], torch.bfloat16, 3, precision=precision)
    lacking[1].grad = None
    for _ in range(2):
        opt.step()
        partial.step()
    assert sorted(partial.state_dict()["state"]) == [0, 2]
    for p, w in zip(params, lacking):
        p.data.copy_(w)
    opt.load_state_dict(torch.load(_saved(partial), weights_only=True))
    assert all(torch.equal(a, b) for a, b in zip(snapshot(params, opt), snapshot(lacking, partial)))


def test_masters_follow_the_weights_where_a_checkpoint_has_none():
    """A torch.optim.AdamW checkpoint with the bf16 weights saved beside it, loaded after the state was made from others."""
    source, _ = make([5000, 300], torch.bfloat16, 4)
    ref = torch.optim.AdamW(source, lr=1e-3)
    ref.step()
    params, opt = make([5000, 300], torch.bfloat16, 3, precision="fp32")
    opt.step()
    for p, s in zip(params, source):
        p.data.copy_(s)
    opt.load_state_dict(ref.state_dict())
    for i, s in enumerate(source):
        assert torch.equal(opt.arenas[0].master_of(i), s.detach().float())
    assert opt.arenas[0].steps.tolist() == [1, 1]
    for group in opt.param_groups:
        group.update(lr=0.0)
    opt.step()
    assert all(torch.equal(p, s) for p, s in zip(params, source))


@pytest.mark.parametrize("change, message", [
    (dict(betas=(1.5, 0.9)), "betas"), (dict(lr=-1.0), "learning rate"), (dict(eps=-1.0), "epsilon"),
    (dict(weight_decay=float("nan")), "weight_decay"), (dict(maximize=True), "maximize"), (dict(amsgrad=True), "amsgrad"),
    (dict(lr=torch.zeros(2)), "lr must be"), (dict(decoupled_weight_decay=False), "decoupled"), (dict(eps=None), "no eps")])
def test_checkpoint_settings_that_it_cannot_follow_are_refused(change, message):
    """Nothing changes, the learning rate's tensor included."""
    lr = torch.full((1,), 1e-3, device="cuda")
    params, opt = make([300], torch.bfloat16, 3, lr=lr)
    opt.step()
    saved = opt.state_dict()
    saved["param_groups"][0].update(change)
    if "eps" in change and change["eps"] is None:
        del saved["param_groups"][0]["eps"]
    before, group = snapshot(params, opt), dict(opt.param_groups[0])
    with pytest.raises((ValueError, TypeError), match=message):
        opt.load_state_dict(saved)
    assert all(torch.equal(a, b) for a, b in zip(before, snapshot(params, opt)))
    after = opt.param_groups[0]
    assert after["lr"] is lr and float(lr) == pytest.approx(1e-3)
    assert all(after[k] == group[k] for k in ("betas", "eps", "weight_decay"))


# --------------------------------------------------------------------------- refusals

def test_refusals():
    params, opt = make([300], torch.bfloat16, 1)
    opt.step()
    with pytest.raises(TypeError, match="grad_scale"):
        opt.step(grad_scale=torch.ones(1))
    with pytest.raises(TypeError, match="found_inf"):
        opt.step(found_inf=torch.ones(2, device="cuda"))
    opt.clip_grad_norm_(1.0)
    with pytest.raises(ValueError, match="clip coefficient"):
        opt.step(grad_scale=torch.ones(1, device="cuda"))
    params[0].data = params[0].data[:100].clone()
    with pytest.raises(RuntimeError, match="changed after"):
        params[0].grad = params[0].grad[:100].clone()
        opt.step()
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ab.GraphAdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float16, device="cuda"))]).prepare()
    with pytest.raises(ValueError, match="non-contiguous"):
        ab.GraphAdamW([torch.nn.Parameter(torch.zeros(4, 4, device="cuda").t()[1:])]).prepare()
    assert int(opt.arenas[0].steps[0]) == 1


def test_past_32_bits():
    """A tensor of more than 2^32 values: its first and last blocks equal those of a short tensor with the same values."""
    n, tail = 2 ** 32 + 1000, 4096 + 1000
    if torch.cuda.get_device_properties(0).total_memory < 80 << 30:
        pytest.skip("needs 80 GB")
    torch.cuda.empty_cache()
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    values, grads = (torch.empty(tail, device="cuda").normal_(generator=gen).bfloat16() for _ in range(2))
    p.data[-tail:] = values
    p.grad[-tail:] = grads
    opt = ab.GraphAdamW([p], **HYPER, precision="int8", stochastic_rounding=False)
    opt.step()
    short = torch.nn.Parameter(values.clone())
    short.grad = grads
    ab.GraphAdamW([short], **HYPER, precision="int8", stochastic_rounding=False).step()
    assert torch.equal(p.detach()[-tail:], short)
    assert float(p.detach()[:-tail].abs().max()) == 0.0
    del opt, p
    torch.cuda.empty_cache()
