"""The optimizer operators on a fusion plan, against a plain 64-bit implementation.

Tolerances count roundings of u = 2^-24 (fp32, half a step relative) and of the stored type's half step.
Norm: fp64 (whose roundings are 2^-29 u each) but for the result's rounding: 1.01 u.  The clip coefficient takes the rounded norm
and is rounded itself: 2.02 u.
AdamW, with d(.) for an error bound: g' = scale g: u |g'|.  m: two products with rounded constants and one sum: 4 u (|b1 m| +
|(1 - b1) g'|).  v: the square has 3 u (g' twice, the product), the products with rounded constants 2 u each, the sum 1: 6 u v.
root = sqrt(v) * c + eps: v's 6 u halved, sqrt 2 u (1 ulp), c rounded and multiplied 2 u, eps rounded and added 2 u: 9 u.
update = m / root * s: the division 3 u (1 ulp or better), s rounded and multiplied 2 u: 14 u |update| + d(m) / m * |update|.
w = w * decay - update: decay rounded, multiplied, subtracted: 3 u |w| + 1 u |update|.  The fp32 result is what is held in a
master or an fp32 weight; a 16-bit weight is off by half a step more."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BLOCK = 256
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


@pytest.fixture(scope="module")
def comp():
    import torch
    assert torch.cuda.is_available(), "needs a GPU"
    import oneccl_amd.comp as c
    c.lib()
    return c


def code(comp, kind):
    return {"float32": comp.FLOAT32, "bfloat16": comp.BFLOAT16, "float16": comp.FLOAT16}[kind]


# counts: one element; nothing but odd sizes and an empty tensor; more tensors than one launch's table; whole items and their edges
GROUPS = {
    "one": [1],
    "odd": [3, 0, 257, 1, 8191, 70001, 255, 256, 511, 0, 4099],
    "many": [int(c) for c in np.exp(np.random.RandomState(1).uniform(0, 8, 600))],
    "items": [8192, 8193, 16384, 4096, 2048, 2049, 24575],
    "large": [2500000, 77, 1300001],
}


class Case:
    """A plan with parameters (a list, each at an address of its own), gradients in both forms, and states, all seeded."""

    def __init__(self, comp, counts, param="float32", grad="float32", master=False, eight=False, align=1, shift=0, seed=0, grad_scale=1e-3):
        import torch
        rng = np.random.default_rng(seed)
        self.comp, self.counts, self.eight = comp, counts, eight
        if eight:
            align = BLOCK * SIZE[grad]
        self.plan = comp.FusionPlan(counts, code(comp, grad), align)
        self.first = [self.plan.offset(i) // SIZE[grad] for i in range(len(counts))]
        self.n = self.plan.elements
        self.inside = np.zeros(self.n, bool)
        for f, c in zip(self.first, counts):
            self.inside[f:f + c] = True

        def put(values, kind):                   # starts `shift` elements into its memory
            t = torch.zeros(len(values) + shift + 1, dtype=getattr(torch, kind), device="cuda")
            t[shift:shift + len(values)] = torch.from_numpy(np.asarray(values, np.float32)).to(getattr(torch, kind)).cuda()
            return t[shift:shift + len(values)]
        w = (0.02 * rng.standard_normal(self.n)).astype(np.float32)
        g = (grad_scale * rng.standard_normal(self.n) * rng.standard_normal(self.n)).astype(np.float32)
        self.params = [put(w[f:f + c], param) for f, c in zip(self.first, counts)]
        self.buffer = put(g, grad)
        self.grads = [put(g[f:f + c], grad) for f, c in zip(self.first, counts)]
        self.master = put(w, "float32") if master else None
        m, v = (3e-4 * rng.standard_normal(self.n)).astype(np.float32), ((5e-4 * rng.standard_normal(self.n)) ** 2).astype(np.float32)
        if eight:
            self.m, self.v = (torch.zeros(self.n, dtype=torch.uint8, device="cuda") for _ in range(2))
            self.scales = torch.zeros(2 * -(-self.n // BLOCK), dtype=torch.uint8, device="cuda")
            self.plan.state_encode(put(m, "float32"), put(v, "float32"), self.m, self.v, self.scales)
        else:
            self.m, self.v, self.scales = put(m, "float32"), put(v, "float32"), None

    def values(self):
        """Weights (fp32 where there is a master), states and gradients as float64, in the plan's layout."""
        import torch
        w = np.zeros(self.n)
        for f, c, p in zip(self.first, self.counts, self.params):
            w[f:f + c] = p.cpu().double().numpy()
        if self.master is not None:
            w = np.where(self.inside, self.master.cpu().double().numpy(), w)
        if self.eight:
            m, v = (torch.zeros(self.n, device="cuda") for _ in range(2))
            self.plan.state_decode(self.m, self.v, self.scales, m, v)
        else:
            m, v = self.m, self.v
        m, v, g = (np.where(self.inside, x.cpu().double().numpy(), 0.0) for x in (m, v, self.buffer))
        return np.where(self.inside, w, 0.0), m, v, g

    def step(self, buffer=False, **kw):
        self.plan.adamw(self.params, self.buffer if buffer else self.grads, self.m, self.v, scales=self.scales, master=self.master, **kw)


def adamw(w, m, v, g, lr, beta1, beta2, eps, weight_decay, step, scale=1.0):
    """The step in 64 bits, and the bounds of the fp32 step's errors (weights, m, v)."""
    g = g * scale
    m1, m2 = beta1 * m, (1 - beta1) * g
    m, v = m1 + m2, beta2 * v + (1 - beta2) * g * g
    dm, dv = 4 * U * (np.abs(m1) + np.abs(m2)) + 2.0 ** -149, 6 * U * v + 2.0 ** -148
    root = np.sqrt(v) / math.sqrt(1 - beta2 ** step) + eps
    s = lr / (1 - beta1 ** step)
    update = m / root * s
    x = w * (1 - lr * weight_decay) - update
    return x, m, v, 3 * U * np.abs(w) + 15 * U * np.abs(update) + dm / root * s, dm, dv


HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=3)


def half_step(kind, x):
    import torch
    info = torch.finfo(getattr(torch, kind))
    return np.abs(x) * info.eps / 2 + info.smallest_normal * info.eps / 2


def state_steps(x, unit, smallest, mantissa):
    """Distance of the values around |x| that the 8-bit format has: `smallest` is its smallest normal value in units."""
    e = np.floor(np.log2(np.maximum(np.abs(x) / unit, smallest)))
    return 2.0 ** (e - mantissa) * unit


def check_states(c, m, v, dm, dv, m_ref, v_ref, steps):
    """8-bit states are within `steps` of the format's distances (1/2: nearest) around the exact ones, plus the fp32 errors; the
    distance is taken a little above, where the next power of two begins."""
    unit = 2.0 ** (c.scales.cpu().numpy().astype(np.float64).reshape(-1, 2) - 127)
    um, uv = (np.repeat(unit[:, i], BLOCK)[:c.n] for i in (0, 1))
    assert (np.abs(m - m_ref) <= steps * state_steps(np.abs(m_ref) + dm, um, 2.0 ** -6, 3) + dm)[c.inside].all()
    close = np.abs(v - v_ref) <= steps * state_steps(v_ref + dv, uv, 16.0, 4) + dv
    least = (v == uv) & (v_ref > 0) & (v_ref <= uv)                    # what is above zero stays so
    assert (close | least)[c.inside].all()
    assert not ((v == 0) & (v_ref > dv))[c.inside].any()


COMBOS = [("float32", "float32", False), ("float32", "bfloat16", False), ("bfloat16", "bfloat16", True), ("bfloat16", "bfloat16", False),
          ("float16", "float16", True), ("float16", "float32", False), ("bfloat16", "float32", True)]


@pytest.mark.parametrize("group", list(GROUPS))
@pytest.mark.parametrize("param,grad,master", COMBOS)
@pytest.mark.parametrize("state", ["32", "8", "8 stochastic"])
def test_adamw(comp, group, param, grad, master, state):
    import torch
    c = Case(comp, GROUPS[group], param, grad, master, state != "32", shift=1 if group == "odd" and state == "32" else 0, seed=len(group))
    scale = torch.tensor(0.37, device="cuda")
    w, m, v, g = c.values()
    before = [t.clone() for t in ([c.m, c.v] + ([c.master] if master else []))]
    kw = dict(HYPER, grad_scale=scale, seed=99 if state == "8 stochastic" else None)
    c.step(buffer=group in ("many", "items"), **kw)
    x, m_ref, v_ref, dx, dm, dv = adamw(w, m, v, g, scale=float(scale), **HYPER)
    w1, m1, v1, _ = c.values()
    hold = half_step(param, np.abs(x) + dx) if param != "float32" else 0.0
    assert (np.abs(w1 - x) <= dx + (0.0 if master else hold))[c.inside].all()
    for f, n, p in zip(c.first, c.counts, c.params):                 # the weights are the master's rounding
        if master:
            assert torch.equal(p, c.master[f:f + n].to(p.dtype))
    if state == "32":
        assert (np.abs(m1 - m_ref) <= dm)[c.inside].all() and (np.abs(v1 - v_ref) <= dv)[c.inside].all()
    else:
        check_states(c, m1, v1, dm, dv, m_ref, v_ref, 0.5 if state == "8" else 1.0)
    out = torch.from_numpy(~c.inside).cuda()
    for t, b in zip([c.m, c.v] + ([c.master] if master else []), before):
        assert torch.equal(t[out], b[out]), "written between the tensors"


@pytest.mark.parametrize("eight", [False, True])
def test_forms_of_the_gradients_and_device_scalars_agree(comp, eight):
    """Tensor by tensor or from the buffer, step and learning rate from the host or from the device: the same bits (the learning
    rate is a float on the device, so the host's call takes the same float)."""
    import torch
    lr = float(np.float32(3e-3))
    runs = []
    for k in range(3):
        c = Case(comp, GROUPS["odd"], "bfloat16", "bfloat16", True, eight, seed=4)
        kw = dict(beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.05, seed=7 if eight else None)
        if k < 2:
            c.step(buffer=k == 1, lr=lr, step=1000, **kw)
        else:
            c.step(lr=123.0, step=1, lr_ptr=torch.tensor([lr], device="cuda"), step_ptr=torch.tensor([1000], device="cuda"), **kw)
        runs.append([c.master, c.m, c.v] + c.params)
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("eight", [False, True])
def test_no_step_for_a_factor_that_is_not_finite(comp, eight):
    import torch
    for bad in (math.nan, math.inf, -math.inf):
        c = Case(comp, GROUPS["odd"], eight=eight)
        before = [t.clone() for t in [c.m, c.v] + c.params]
        c.step(grad_scale=torch.tensor([bad], device="cuda"), **HYPER)
        for a, b in zip([c.m, c.v] + c.params, before):
            assert torch.equal(a, b)


@pytest.mark.parametrize("eight", [False, True])
def test_a_gradient_that_is_not_finite_reaches_its_own_element_alone(comp, eight):
    import torch
    c, clean = (Case(comp, [700, 300], eight=eight, seed=2) for _ in range(2))
    where = [(0, 5), (0, 260), (1, 299)]
    for (t, i), x in zip(where, (math.nan, math.inf, -math.inf)):
        c.grads[t][i] = x
        clean.grads[t][i] = 0.0                  # takes the element out of its block's largest value
    hit = torch.zeros(c.n, dtype=torch.bool, device="cuda")
    for t, i in where:
        hit[c.first[t] + i] = True
    for x in (c, clean):
        x.step(**HYPER)
    w, m, v, _ = c.values()
    mask = hit.cpu().numpy()
    assert np.isnan(w[mask]).all() and not np.isfinite(v[mask]).any() and not np.isfinite(m[mask]).any()
    assert np.isfinite(w[~mask]).all() and np.isfinite(m[~mask]).all() and np.isfinite(v[~mask]).all()
    w2, m2, v2, _ = clean.values()
    assert np.array_equal(w[~mask], w2[~mask])


@pytest.mark.parametrize("grad", ["float32", "bfloat16"])
def test_the_smallest_gradients_and_eps(comp, grad):
    """Second moments that are denormal (gradients from 1e-22 to 1e-17) with an eps that they matter beside, and weights without
    any gradient: nothing becomes infinite or NaN, and the update is the formula's (m and v of a first step are exact multiples;
    their denormal values are off by half of 2^-149, which the root of v feels as sqrt(2^-149) at most)."""
    import torch
    n = 3000
    plan = comp.FusionPlan([n], code(comp, grad), 1)
    g = torch.zeros(n, dtype=getattr(torch, grad), device="cuda")
    g[1000:] = torch.logspace(-22, -17, 2000, device="cuda").to(g.dtype)
    p, m, v = (torch.zeros(plan.elements, device="cuda") for _ in range(3))
    eps = 1e-20
    plan.adamw([p], [g], m, v, lr=1.0, beta1=0.9, beta2=0.95, eps=eps, weight_decay=0.0, step=1)
    assert not p[:1000].any() and torch.isfinite(p).all()
    x = g[1000:].double().cpu().numpy()
    want = -x / (x + eps)
    root_off = math.sqrt(2.0 ** -149 / 0.05)                            # sqrt(v + 2^-149) - sqrt(v) is at most sqrt(2^-149)
    tol = 20 * U + root_off / (x + eps) + 2.0 ** -149 / 0.1 / (x + eps)
    assert (np.abs(p[1000:].double().cpu().numpy() - want) <= tol).all()


def test_a_fresh_state_and_zero_gradients(comp):
    """All-zero 8-bit states; a zero gradient moves a weight by its decay alone, states stay zero."""
    import torch
    c = Case(comp, GROUPS["odd"], eight=True)
    for t in (c.m, c.v, c.scales):
        t.zero_()
    for g in c.grads:
        g.zero_()
    c.grads[2][7] = 1e-3
    w, _, _, _ = c.values()
    c.step(**dict(HYPER, step=1))
    w1, m, v, _ = c.values()
    at = c.first[2] + 7
    rest = c.inside.copy()
    rest[at] = False
    assert (np.abs(w1 - w * (1 - 1e-3)) <= 2 * U * np.abs(w))[rest].all() and not m[rest].any() and not v[rest].any()
    assert abs(w1[at] - (w[at] * (1 - 1e-3) - 1e-2 * 1e-3 / (1e-3 + 1e-8))) <= 32 * U * 1e-2


# ---- 8-bit states ------------------------------------------------------------------------------------------------------

def books():
    m = np.array([(c % 8) * 2.0 ** -9 if c < 8 else (8 + c % 8) * 2.0 ** (c // 8 - 10) for c in range(127)] + [np.nan])
    v = np.array([float(c) if c < 16 else (16 + c % 16) * 2.0 ** (c // 16 - 1) for c in range(255)] + [np.nan])
    return m, v


def test_every_code_and_scale(comp):
    """All codes under every scale byte from 1 to 247 (the largest that an encoding gives), as fp32: exact."""
    import torch
    book_m, book_v = books()
    blocks = 247
    plan = comp.FusionPlan([BLOCK] * blocks, comp.FLOAT32, 4 * BLOCK)
    codes = torch.arange(256, device="cuda", dtype=torch.int32).to(torch.uint8).repeat(blocks)
    scales = torch.arange(1, blocks + 1, dtype=torch.int32, device="cuda").to(torch.uint8).repeat_interleave(2)
    m, v = (torch.zeros(plan.elements, device="cuda") for _ in range(2))
    plan.state_decode(codes, codes, scales, m, v)
    s = 2.0 ** (np.arange(1, blocks + 1) - 127.0)
    with np.errstate(over="ignore"):                                   # 448 * 2^120 is beyond fp32: infinite
        want_m = (np.concatenate([book_m, -book_m])[None] * s[:, None]).reshape(-1).astype(np.float32)
        want_v = (book_v[None] * s[:, None]).reshape(-1).astype(np.float32)
    assert np.array_equal(m.cpu().numpy(), want_m, equal_nan=True)
    assert np.array_equal(v.cpu().numpy(), want_v, equal_nan=True)
    # and what is decoded is encoded as it was, where a block's scale can be (its codes reach the top of the format)
    m2, v2, s2 = torch.zeros_like(codes), torch.zeros_like(codes), torch.zeros_like(scales)
    few = 230                                                          # exp_avg_sq is finite under these
    plan.state_encode(m, torch.where(torch.isfinite(v) | torch.isnan(v), v, torch.zeros_like(v)), m2, v2, s2)
    n = few * BLOCK
    assert torch.equal(v2[:n], codes[:n]) and torch.equal(s2[:2 * few], scales[:2 * few])
    c = codes[:n].clone()
    same = m2[:n] == c
    nan = (c & 127) == 127
    assert (same | nan).all() and ((m2[:n] & 127) == 127)[nan].all()


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_encode_to_nearest(comp, kind):
    """Scales and codes by the definition, to the bit: values over many decades, exact ties, zeros, values that are not finite."""
    import torch
    rng = np.random.default_rng(3)
    counts = [1, 255, 256, 257, 5000, 90001]
    plan = comp.FusionPlan(counts, comp.BFLOAT16, 2 * BLOCK)
    n = -(-plan.elements // BLOCK) * BLOCK                             # whole blocks, the last one's rest is outside
    book_m, book_v = books()
    first = [plan.offset(i) // 2 for i in range(len(counts))]
    inside = np.zeros(n, bool)
    for f, c in zip(first, counts):
        inside[f:f + c] = True
    block_scale = np.repeat(2.0 ** rng.integers(-120, 90, n // BLOCK), BLOCK)
    m = rng.standard_normal(n) * 10.0 ** rng.uniform(-6, 0, n) * block_scale
    v = rng.standard_normal(n) ** 2 * 10.0 ** rng.uniform(-8, 0, n) * block_scale
    tie = rng.random(n) < 0.2
    i, j = rng.integers(0, 126, n), rng.integers(0, 254, n)
    m[tie] = ((book_m[i] + book_m[i + 1]) / 2 * block_scale)[tie]      # halves of the grid wherever the block's scale is a power of two
    v[tie] = ((book_v[j] + book_v[j + 1]) / 2 * block_scale)[tie]
    for p, x in ((0.02, 0.0), (0.01, np.nan), (0.01, np.inf), (0.01, -np.inf)):
        at = rng.random(n) < p
        m[at], v[at] = x, abs(x)
    m[first[3]:first[3] + 257] = 0.0                                   # a block of zeros
    v[first[3]:first[3] + 257] = np.nan                                # a block with nothing finite
    v[first[4] + 3] = -1.0
    tm, tv = (torch.from_numpy(x.astype(np.float32)).to(getattr(torch, kind)).cuda() for x in (m, v))
    m, v = tm.cpu().double().numpy(), tv.cpu().double().numpy()
    cm, cv = (torch.full((n,), 77, dtype=torch.uint8, device="cuda") for _ in range(2))
    sc = torch.full((2 * (n // BLOCK),), 88, dtype=torch.uint8, device="cuda")
    plan.state_encode(tm, tv, cm, cv, sc)
    for x, book, top, got, scale, signed in ((m, book_m, 448.0, cm, sc[0::2], True), (v, book_v, 30 * 2.0 ** 14, cv, sc[1::2], False)):
        mag = np.where(inside & np.isfinite(x), np.abs(x), 0.0).reshape(-1, BLOCK)
        largest = mag.max(1)
        s = np.ones(len(largest), np.int64)
        for b, l in enumerate(largest):
            while l > top * 2.0 ** (s[b] - 127):
                s[b] += 1
        assert np.array_equal(scale.cpu().numpy().astype(np.int64), s)
        y = mag.reshape(-1) / np.repeat(2.0 ** (s - 127.0), BLOCK)
        values = book[:-1]
        lo = np.clip(np.searchsorted(values, y, side="right") - 1, 0, len(values) - 2)
        up, down = values[lo + 1] - y, y - values[lo]
        want = np.where((up < down) | ((up == down) & (lo % 2 == 1)), lo + 1, lo)
        if not signed:
            want = np.where((want == 0) & (x > 0), 1, want)
        bad = ~np.isfinite(x) | (~np.bool_(signed) & (x < 0))
        want = np.where(bad, 127 if signed else 255, want)
        g = got.cpu().numpy().astype(np.int64)
        assert (g[~inside] == 77).all()
        if signed:
            assert (((g & 127) == want) & (((g >> 7) == np.signbit(x)) | np.isnan(x)))[inside].all()
        else:
            assert (g == want)[inside].all()


def test_stochastic_rounding_has_no_bias(comp):
    """States that lie between two codes of their block (whose scale one large element fixes): after a step with no gradient and
    beta = 1 - 2^-10 every element goes up with the probability of its distance.  The mean of n = 65,024 draws of variance <= 1/4
    is off by at most 6 sqrt(1 / 4n) in all but 2e-9 of all seeds (the seed is fixed), plus the 2^-17 by which 16 random bits
    cut off what is below them, and the next step with the same seed draws others."""
    import torch
    n = 256 * 256
    draws = []
    for step in (5, 6):
        plan = comp.FusionPlan([n], comp.FLOAT32, 4 * BLOCK)
        m, v, p, g = (torch.zeros(n, device="cuda") for _ in range(4))
        m[:], v[:] = 13.0, 24.0
        m[::256], v[::256] = 448.0, 30.0 * 2 ** 14
        cm, cv, sc = torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(2 * n // BLOCK, dtype=torch.uint8, device="cuda")
        plan.state_encode(m, v, cm, cv, sc)
        b = 1 - 2.0 ** -4
        plan.adamw([p], [g], cm, cv, scales=sc, lr=0.0, beta1=b, beta2=b, eps=1.0, weight_decay=0.0, step=step, seed=12345)
        plan.state_decode(cm, cv, sc, m, v)
        unit = 2.0 ** (sc.cpu().numpy().astype(int) - 127.0)
        assert (unit == 1).all()
        rest = torch.arange(n, device="cuda") % 256 != 0
        for x, exact, lo, hi in ((m[rest], 13 * b, 12.0, 13.0), (v[rest], 24 * b, 22.0, 23.0)):
            up = (x == hi).double()
            assert ((x == hi) | (x == lo)).all()
            share = (exact - lo) / (hi - lo)
            assert abs(float(up.mean()) - share) <= 6 * math.sqrt(0.25 / up.numel()) + 2.0 ** -17
            draws.append(up)
    # m against v, and one step against the next: independent draws agree as often as their shares say
    for a, b_ in ((draws[0], draws[1]), (draws[0], draws[2]), (draws[1], draws[3])):
        cov = float((a * b_).mean() - a.mean() * b_.mean())
        assert abs(cov) <= 6 * 0.25 / math.sqrt(a.numel())


# ---- norm --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("group", list(GROUPS))
@pytest.mark.parametrize("grad", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("align,shift", [(1, 0), (1, 1), (512, 0)])
def test_norm(comp, group, grad, align, shift):
    import torch
    c = Case(comp, GROUPS[group], "float32", grad, align=align, shift=shift, seed=11, grad_scale=0.3)
    c.buffer[torch.from_numpy(~c.inside).cuda()] = math.nan              # padding is no gradient
    exact = math.sqrt(sum(float((g.double() ** 2).sum()) for g in c.grads))
    for mult, most in ((1.0, 0.0), (0.125, 1e-2), (-0.5, 1e9), (2.0, exact)):
        results = []
        for grads in (c.grads, c.buffer):
            r = torch.full((2,), 7.0, device="cuda")
            c.plan.norm(grads, r, multiplier=mult, max_norm=most)
            norm, coef = r.tolist()
            assert abs(norm - abs(mult) * exact) <= 1.01 * U * abs(mult) * exact
            want = mult * min(1.0, most / (abs(mult) * exact + 1e-6)) if most > 0 else mult
            assert abs(coef - want) <= 2.02 * U * abs(want)
            again = torch.zeros(2, device="cuda")
            c.plan.norm(grads, again, multiplier=mult, max_norm=most)
            assert torch.equal(r, again)
            results.append(r)


def test_norm_of_nothing_and_of_what_is_not_finite(comp):
    import torch
    plan = comp.FusionPlan([0, 0], comp.FLOAT32, 1)
    r = torch.full((2,), 7.0, device="cuda")
    plan.norm([torch.zeros(0, device="cuda")] * 2, r, multiplier=3.0, max_norm=1.0)
    assert r.tolist() == [0.0, 3.0]
    for x in (math.nan, math.inf, -math.inf, 3e38):
        c = Case(comp, GROUPS["odd"])
        c.grads[3][0] = x
        c.plan.norm(c.grads, r, multiplier=2.0, max_norm=1.0)          # 6e38 is no float
        assert not math.isfinite(r[0].item()) and math.isnan(r[1].item())
        before = [p.clone() for p in c.params]
        c.step(grad_scale=r[1:], **HYPER)
        assert all(torch.equal(a, b) for a, b in zip(before, c.params))


@pytest.mark.parametrize("grad", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", [2.0 ** -140, 2.0 ** -100, 2.0 ** 80, 2.0 ** 120])
def test_norm_of_gradients_whose_squares_no_float_holds(comp, grad, size):
    import torch
    c = Case(comp, GROUPS["odd"], "float32", grad, seed=12, grad_scale=0.3)
    for g in c.grads:
        g.copy_((g.double() * size).to(g.dtype))                          # denormals for the smallest; zeros in bfloat16
    exact = math.sqrt(sum(float((g.double() ** 2).sum()) for g in c.grads))
    r = torch.zeros(2, device="cuda")
    c.plan.norm(c.grads, r, max_norm=1.0)
    norm, coef = r.tolist()
    # a norm or a coefficient below the normal range is off by half a denormal's step
    assert abs(norm - exact) <= 1.01 * U * exact + 2.0 ** -150
    want = min(1.0, 1.0 / (exact + 1e-6))
    assert abs(coef - want) <= 2.02 * U * want + 2.0 ** -150


def test_refusals(comp):
    import torch
    c = Case(comp, [300, 5], "bfloat16", "bfloat16", True)
    e = Case(comp, [300, 5], "bfloat16", "bfloat16", True, eight=True)
    refused = (ValueError, comp.CclError)
    for kw in (dict(lr=-1.0), dict(lr=math.nan), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(eps=0.0), dict(eps=1e-40), dict(weight_decay=-1.0), dict(step=0)):
        with pytest.raises(refused):
            c.step(**dict(HYPER, **kw))
    with pytest.raises(refused):
        c.step(lr_ptr=torch.zeros(1, device="cuda"), workspace=torch.zeros(8, dtype=torch.uint8, device="cuda"), **HYPER)
    with pytest.raises(refused):
        c.step(**dict(HYPER, seed=1))                                    # 32-bit states have nothing to round
    for kw in (dict(grad_scale=torch.zeros(1, device="cuda", dtype=torch.float64)), dict(step_ptr=torch.zeros(1, device="cuda")),
               dict(lr_ptr=torch.zeros(1))):
        with pytest.raises(refused):
            c.step(**dict(HYPER, **kw))
    call = c.plan.adamw
    for args in ((c.params[:1], c.grads, c.m, c.v), (c.params, c.grads[:1], c.m, c.v), (c.params, c.grads, c.m[:-1], c.v), (c.params, c.grads, c.m.double(), c.v),
                 (c.params, [g.float() for g in c.grads], c.m, c.v), ([c.params[0][::2], c.params[1]], c.grads, c.m, c.v),
                 (c.params, c.buffer[:-1], c.m, c.v), ([c.params[0].double(), c.params[1].double()], c.grads, c.m, c.v)):
        with pytest.raises(refused):
            call(*args, **HYPER)
    with pytest.raises(refused):
        e.plan.adamw(e.params, e.grads, e.m, e.v, scales=None, **HYPER)
    with pytest.raises(refused):                                         # a tight layout has no blocks
        c.plan.adamw(c.params, c.grads, e.m, e.v, scales=e.scales, **HYPER)
    full = Case(comp, [300, 5])
    with pytest.raises(refused):                                         # fp32 weights need no copy
        full.plan.adamw(full.params, full.grads, full.m, full.v, master=full.m, **HYPER)
    with pytest.raises(refused):
        comp.FusionPlan([4], comp.INT32, 1).norm([torch.zeros(4, dtype=torch.int32, device="cuda")], torch.zeros(2, device="cuda"))
    with pytest.raises(refused):
        c.plan.norm(c.grads, torch.zeros(2, device="cuda"), workspace=torch.zeros(1, dtype=torch.uint8, device="cuda"))
    with pytest.raises(refused):
        c.plan.norm(c.grads, torch.zeros(2, device="cuda"), max_norm=math.nan)
    with pytest.raises(refused):
        e.plan.state_decode(e.m, e.v, e.scales, torch.zeros(e.n, device="cuda").half(), torch.zeros(e.n, device="cuda").half())
    L, o = comp.lib(), comp.AdamwOptions(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, step=1)
    import ctypes as C
    P = comp._ptr_array(c.params)
    args = [c.plan._h, comp.BFLOAT16, P, None, c.buffer.data_ptr(), 0, c.m.data_ptr(), c.v.data_ptr(), None, None, C.byref(o), None]
    o.lr_ptr = c.m.data_ptr()                                            # and nowhere to put what follows from it
    assert L.mi_ccl_fusion_adamw(*args) == comp.INVALID_ARGUMENTS
    o.lr_ptr = None
    for i, x in ((1, comp.INT8), (2, None), (3, P), (4, None), (4, c.buffer.data_ptr() + 1), (5, 2), (6, None), (7, c.v.data_ptr() + 2), (9, c.m.data_ptr() + 1), (10, None)):
        bad = list(args)
        bad[i] = x
        assert L.mi_ccl_fusion_adamw(*bad) == comp.INVALID_ARGUMENTS, i


@pytest.mark.parametrize("eight", [False, True])
def test_offsets_past_32_bits(comp, eight):
    """A group of 2^31 elements and more: bytes of gradients, weights and states past 2^32.  All is zero but pieces at the ends and around
    the elements where a 32-bit offset of bytes or elements would turn over."""
    import torch
    counts = [70001, (1 << 31) + 12345, 4099]
    plan = comp.FusionPlan(counts, comp.BFLOAT16, 2 * BLOCK if eight else 2)
    first, n = [plan.offset(i) // 2 for i in range(3)], plan.elements
    buffer = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    params = [torch.zeros(c, dtype=torch.bfloat16, device="cuda") for c in counts]
    states = [torch.zeros(n, dtype=torch.uint8 if eight else torch.float32, device="cuda") for _ in range(2)]
    scales = torch.zeros(2 * -(-n // BLOCK), dtype=torch.uint8, device="cuda") if eight else None
    gen = torch.Generator("cuda").manual_seed(5)
    pieces = [(0, 0, 5000), (1, 0, 700), (1, (1 << 30) - 777, 1500), (1, (1 << 31) - first[1] - 600, 1111), (1, counts[1] - 800, 800), (2, 0, 4099)]
    for t, e, size in pieces:
        buffer[first[t] + e:first[t] + e + size] = (1e-3 * torch.randn(size, device="cuda", generator=gen)).bfloat16()
        params[t][e:e + size] = (0.02 * torch.randn(size, device="cuda", generator=gen)).bfloat16()
    old = [params[t][e:e + size].double().cpu().numpy() for t, e, size in pieces]
    grads = [buffer[first[t] + e:first[t] + e + size].double().cpu().numpy() for t, e, size in pieces]
    exact = math.sqrt(sum(float((g ** 2).sum()) for g in grads))
    result = torch.zeros(2, device="cuda")
    for source in (buffer, [buffer[f:f + c] for f, c in zip(first, counts)]):
        plan.norm(source, result)
        assert abs(result[0].item() - exact) <= 1.01 * U * exact
    plan.adamw(params, buffer, *states, scales=scales, **HYPER)
    nonzero = sum(int(torch.count_nonzero(p[a:a + (1 << 28)])) for p in params for a in range(0, p.numel(), 1 << 28))
    assert 0 < nonzero <= sum(size for _, _, size in pieces)
    for (t, e, size), w, g in zip(pieces, old, grads):
        x, m, v, dx, dm, dv = adamw(w, 0 * w, 0 * w, g, **HYPER)
        got = params[t][e:e + size].double().cpu().numpy()
        assert (np.abs(got - x) <= dx + half_step("bfloat16", np.abs(x) + dx)).all()
        at = slice(first[t] + e, first[t] + e + size)
        if not eight:
            assert (np.abs(states[0][at].double().cpu().numpy() - m) <= dm).all()
            assert (np.abs(states[1][at].double().cpu().numpy() - v) <= dv).all()
        else:
            assert int(torch.count_nonzero(states[1][at])) == np.count_nonzero(g)       # a second moment above zero stays above it


def test_the_native_pass_over_tensors_is_built(comp):
    comp.FusionPlan([3], comp.FLOAT32, 1)
    assert comp._native
