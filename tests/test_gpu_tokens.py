"""Tokens sorted by expert and back, against a plain 64-bit implementation on the CPU.

Tolerances: a rounding to a type is off by at most half a step, finfo.eps / 2 relative (half of the smallest denormal below
the normal range).  combine adds top_k products in fp32, one rounding each: top_k * 2^-24 * sum |w y| on top.
combine_backward's rows are one fp32 product and one rounding to the type; its dot products add H terms in fp32, in any
order within H * 2^-24 * sum |g y|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def comp():
    import torch
    assert torch.cuda.is_available(), "needs a GPU"
    import oneccl_amd.comp as c
    c.lib()
    return c


def place(ids, experts, align=1, capacity=0):
    """positions, counts, offsets by the definition."""
    flat = ids.reshape(-1)
    pos = np.full(flat.size, -1, np.int64)
    counts, offsets, begin = np.zeros(experts, np.int64), np.zeros(experts + 1, np.int64), 0
    for e in range(experts):
        mine = np.flatnonzero(flat == e)
        if capacity:
            mine = mine[:capacity]
        pos[mine] = begin + np.arange(mine.size)
        counts[e] = mine.size
        begin += -(-mine.size // align) * align
        offsets[e + 1] = begin
    return pos.reshape(ids.shape), counts, offsets


def make_ids(rng, tokens, k, experts, dropped=0.0, wild=False):
    score = rng.standard_normal((tokens, experts)) + 0.7 * rng.standard_normal(experts)
    ids = np.argsort(-score, axis=1)[:, :k] if experts >= k else rng.integers(0, experts, (tokens, k))
    ids = ids.astype(np.int64)
    ids[rng.random(tokens) < dropped] = -1
    if wild:
        ids[rng.random(ids.shape) < 0.1] = experts
        ids[rng.random(ids.shape) < 0.05] = -(1 << 31)
        ids[rng.random(ids.shape) < 0.05] = (1 << 31) - 1
    return ids


def sort(comp, ids, experts, align=1, capacity=0, kind="int32"):
    import torch
    d = torch.from_numpy(ids.astype(kind)).cuda()
    pos = torch.full(ids.shape, -7, dtype=torch.int32, device="cuda")
    counts, offsets = torch.full((experts,), -7, dtype=torch.int32, device="cuda"), torch.full((experts + 1,), -7, dtype=torch.int32, device="cuda")
    comp.token_sort(d, experts, pos, counts, offsets, align=align, capacity=capacity)
    return pos, counts, offsets


@pytest.mark.parametrize("tokens,k,experts,align,capacity,kind", [
    (1, 1, 1, 1, 0, "int32"), (1, 8, 64, 1, 0, "int64"), (3, 2, 5, 4, 0, "int32"), (64, 1, 3, 1, 7, "int32"), (65, 1, 1, 1, 0, "int64"),
    (1000, 3, 17, 16, 0, "int32"), (1024, 8, 256, 1, 0, "int32"), (8192, 1, 257, 8, 5, "int32"), (8193, 1, 1024, 1, 0, "int64"),
    (2049, 4, 128, 128, 0, "int32"), (20000, 6, 60, 1, 1999, "int32"), (7, 300, 2, 1, 0, "int32"), (4096, 1, 7, 1, 0, "int32"), (4097, 1, 7, 4, 0, "int64"), (300001, 8, 1000, 1, 0, "int32"), (0, 4, 9, 8, 0, "int32"),
])
def test_sort(comp, tokens, k, experts, align, capacity, kind):
    rng = np.random.default_rng(tokens + experts)
    ids = make_ids(rng, tokens, k, experts, 0.1, wild=tokens > 10) if tokens < 100000 else rng.integers(-1, experts + 1, (tokens, k))
    got = sort(comp, ids, experts, align, capacity, kind)
    assert comp.token_rows(tokens, k, experts, align, capacity) >= int(got[2][-1])
    for name, g, w in zip(("positions", "counts", "offsets"), got, place(ids, experts, align, capacity)):
        assert np.array_equal(g.cpu().numpy().astype(np.int64), w), name


def test_sort_of_one_expert_and_of_none(comp):
    """Every entry on one expert (ranks beyond 16 bits), and a batch of masked tokens alone."""
    ids = np.full((70000, 2), 3, np.int64)
    for got, w in zip(sort(comp, ids, 8, 64), place(ids, 8, 64)):
        assert np.array_equal(got.cpu().numpy().astype(np.int64), w)
    ids = np.full((20000, 1), -1, np.int64)
    for got, w in zip(sort(comp, ids, 8, 64), place(ids, 8, 64)):
        assert np.array_equal(got.cpu().numpy().astype(np.int64), w)


# tokens, top_k, experts, hidden, align, dropped: one token, rows of less than a vector, odd rows, more choices than a group of 8
SHAPES = [(1, 8, 64, 4096, 1, 0.0), (1, 1, 1, 1, 1, 0.0), (2, 2, 4, 7, 4, 0.0), (5, 3, 7, 513, 1, 0.3), (33, 2, 16, 64, 16, 0.2), (300, 4, 9, 1031, 8, 0.1),
          (17, 11, 12, 130, 1, 0.0), (3, 1, 2, 20001, 1, 0.0), (600, 2, 128, 264, 128, 0.5), (4, 2, 3, 8, 1, 1.0)]
TYPES = ["float32", "bfloat16", "float16"]


def rows_of(rng, n, hidden, kind, pad=0, shift=0):
    """A [n, hidden] matrix on the device whose rows are `pad` elements apart and start `shift` elements into the memory."""
    import torch
    base = torch.zeros(shift + n * (hidden + pad) + 8, dtype=getattr(torch, kind), device="cuda")
    m = base[shift:shift + n * (hidden + pad)].view(n, hidden + pad)[:, :hidden]
    m.copy_(torch.from_numpy(rng.standard_normal((n, hidden)).astype(np.float32)))
    return m, base


def host(t):
    return t.detach().cpu().double().numpy()


def half_step(kind, x):
    import torch
    info = torch.finfo(getattr(torch, kind))
    return np.abs(x) * info.eps / 2 + info.smallest_normal * info.eps / 2


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("pad,shift", [(0, 0), (3, 1)])
@pytest.mark.parametrize("ordered", [False, True])
def test_dispatch_combine_and_gradients(comp, shape, kind, pad, shift, ordered):
    """Token by token, and in the order of the rows, which large calls take (forced here by the variant knob)."""
    comp.set_param("variant", 8 if ordered else 0)
    try:
        run_dispatch_combine_and_gradients(comp, shape, kind, pad, shift, ordered)
    finally:
        comp.set_param("variant", 0)


def run_dispatch_combine_and_gradients(comp, shape, kind, pad, shift, ordered):
    import torch
    tokens, k, experts, hidden, align, dropped = shape
    rng = np.random.default_rng(hidden)
    ids = make_ids(rng, tokens, k, experts, dropped)
    pos, counts, offsets = sort(comp, ids, experts, align)
    hp, hc, ho = place(ids, experts, align)
    rows = comp.token_rows(tokens, k, experts, align) + 3
    x, _ = rows_of(rng, tokens, hidden, kind, pad, shift)
    out, out_all = rows_of(rng, rows, hidden, kind, pad, shift)
    before = out.clone()
    guard = out_all.clone()
    comp.token_dispatch(x, pos, counts, offsets, out)
    assert comp.last_kernel() == ("token_dispatch_ordered_kernel" if ordered else "token_dispatch_kernel")
    want = host(before)
    want[:ho[-1]] = 0
    for t in range(tokens):
        for j in range(k):
            if hp[t, j] >= 0:
                want[hp[t, j]] = host(x[t])
    assert np.array_equal(host(out), want)                           # a copy: to the bit, rows behind the last as they were
    out.copy_(before)
    assert torch.equal(out_all, guard), "written between the rows"

    y, _ = rows_of(rng, rows, hidden, kind, pad, shift)
    hy = host(y)
    for weighted in (True, False):
        w = torch.from_numpy(rng.standard_normal((tokens, k)).astype(np.float32)).cuda() if weighted else None
        hw = host(w) if weighted else np.ones((tokens, k))
        some = hp >= 0
        terms = np.where(some[:, :, None], hw[:, :, None] * hy[np.maximum(hp, 0)], 0.0)
        res, res_all = rows_of(rng, tokens, hidden, kind, pad, shift)
        keep, guard = res.clone(), res_all.clone()
        comp.token_combine(y, pos, w, res)
        ref = terms.sum(1)
        err = np.abs(host(res) - ref)
        tol = k * U32 * np.abs(terms).sum(1)
        assert (err <= half_step(kind, np.abs(ref) + tol) + tol).all(), err.max()
        res.copy_(keep)
        assert torch.equal(res_all, guard), "written between the rows"

        g, _ = rows_of(rng, tokens, hidden, kind, pad, shift)
        hg = host(g)
        gy, gy_all = rows_of(rng, rows, hidden, kind, pad, shift)
        keep, guard = gy.clone(), gy_all.clone()
        gw = torch.full((tokens, k), 7.0, device="cuda")
        comp.token_combine_backward(g, y, pos, w, counts, offsets, gy, gw)
        assert comp.last_kernel() == ("token_backward_ordered_kernel" if ordered else "token_combine_backward_kernel")
        ref, tol = host(keep), np.zeros((rows, hidden))
        ref[:ho[-1]] = 0
        for t in range(tokens):
            for j in range(k):
                if some[t, j]:
                    ref[hp[t, j]] = hw[t, j] * hg[t]
                    tol[hp[t, j]] = U32 * np.abs(ref[hp[t, j]]) + half_step(kind, ref[hp[t, j]]) * (1 + 1e-6)
        assert (np.abs(host(gy) - ref) <= tol).all()
        dots = np.where(some[:, :, None], hg[:, None, :] * hy[np.maximum(hp, 0)], 0.0)
        assert (np.abs(host(gw) - dots.sum(2)) <= hidden * U32 * np.abs(dots).sum(2)).all()
        # without the weights' gradient: the same rows, y is not looked at
        again = gy.clone()
        gy.copy_(keep)
        comp.token_combine_backward(g, None, pos, w, counts, offsets, gy)
        assert torch.equal(gy, again)
        gy.copy_(keep)
        assert torch.equal(gy_all, guard), "written between the rows"
        gx, _ = rows_of(rng, tokens, hidden, kind, pad, shift)
        comp.token_dispatch_backward(y, pos, gx)
        if not weighted:
            assert torch.equal(gx, (lambda r: (comp.token_combine(y, pos, None, r), r)[1])(torch.zeros_like(gx)))


@pytest.mark.parametrize("variant", [0, 8])
def test_one_expert_twice_and_positions_outside(comp, variant):
    """A token that names an expert twice has two rows there; positions outside the buffer count as none."""
    comp.set_param("variant", variant)
    try:
        run_one_expert_twice_and_positions_outside(comp)
    finally:
        comp.set_param("variant", 0)


def run_one_expert_twice_and_positions_outside(comp):
    import torch
    ids = np.array([[2, 2], [2, 0]], np.int64)
    pos, counts, offsets = sort(comp, ids, 3)
    assert pos.tolist() == [[1, 2], [3, 0]]
    x = torch.arange(1, 3, device="cuda").float()[:, None].expand(2, 5).contiguous()
    out = torch.zeros(4, 5, device="cuda")
    comp.token_dispatch(x, pos, counts, offsets, out)
    assert out[:, 0].tolist() == [2, 1, 1, 2]
    bad = torch.tensor([[4, 1], [-5, 1 << 30]], dtype=torch.int32, device="cuda")
    res = torch.full((2, 5), 9.0, device="cuda")
    comp.token_combine(out, bad, None, res)
    assert res[:, 0].tolist() == [1, 0]
    out2 = torch.full((4, 5), 9.0, device="cuda")
    comp.token_dispatch(x, bad, torch.zeros_like(counts), torch.zeros_like(offsets), out2)
    assert out2[:, 0].tolist() == [9, 1, 9, 9]
    gy, gw = torch.full((4, 5), 9.0, device="cuda"), torch.full((2, 2), 9.0, device="cuda")
    comp.token_combine_backward(x, out, bad, None, torch.zeros_like(counts), torch.zeros_like(offsets), gy, gw)
    assert gy[:, 0].tolist() == [9, 1, 9, 9] and gw.tolist() == [[0, 5], [0, 0]]
    # no rows at all
    comp.token_combine(torch.zeros(0, 5, device="cuda"), bad, None, res)
    assert not res.any()


@pytest.mark.parametrize("experts", [1, 3, 4, 7])
@pytest.mark.parametrize("variant", [0, 8])
def test_an_odd_number_of_experts_reads_no_further_count(comp, variant, experts):
    """counts and offsets are parts of larger arrays whose next words, taken for one more expert's, would clear every row."""
    import torch
    ids = np.arange(24).reshape(12, 2) % experts
    pos, c, o = sort(comp, ids, experts, 4)
    rows = int(o[-1])
    counts, offsets = torch.full((experts + 2,), -rows, dtype=torch.int32, device="cuda"), torch.full((experts + 3,), rows, dtype=torch.int32, device="cuda")
    counts[:experts], offsets[:experts + 1] = c, o
    counts, offsets = counts[:experts], offsets[:experts + 1]
    x = torch.arange(1, 13, device="cuda").float()[:, None].expand(12, 40).contiguous()
    want = torch.zeros(rows, 40, device="cuda")
    want[pos.long().reshape(-1)] = x.repeat_interleave(2, 0)
    comp.set_param("variant", variant)
    try:
        for _ in range(2):
            out, gy, gw = (torch.full(z, 9.0, device="cuda") for z in ((rows, 40), (rows, 40), (12, 2)))
            comp.token_dispatch(x, pos, counts, offsets, out)
            assert torch.equal(out, want)
            comp.token_combine_backward(x, out, pos, None, counts, offsets, gy, gw)
            assert torch.equal(gy, want)
            assert torch.equal(gw[:, 0], 40 * x[:, 0] ** 2) and torch.equal(gw[:, 1], gw[:, 0])
    finally:
        comp.set_param("variant", 0)


# 70,001 x 4104: more tokens than the grid has blocks for them, whose blocks take a second one; 192, 384 and 512 lanes per row, several column
# tiles per row
@pytest.mark.parametrize("tokens,k,experts,hidden,kind", [(6007, 6, 40, 1000, "bfloat16"), (70001, 1, 8, 257, "float32"), (70001, 1, 8, 4104, "bfloat16"),
                                                             (5003, 7, 13, 1540, "bfloat16"), (9001, 1, 5, 5124, "float16"), (7001, 1, 5, 2565, "float32")])
def test_many_runs_in_order_equal_token_by_token(comp, tokens, k, experts, hidden, kind):
    """From 64 MiB of rows the order is taken by itself (runs on every XCD, a last run that is not full): the same rows as without
    scratch memory, to the bit; the weights' gradients within the bound of their sums."""
    import torch
    rng = np.random.default_rng(tokens)
    ids = make_ids(rng, tokens, k, experts, 0.05)
    pos, counts, offsets = sort(comp, ids, experts, 8)
    rows = comp.token_rows(tokens, k, experts, 8)
    t = getattr(torch, kind)
    x = torch.randn(tokens, hidden, device="cuda").to(t)
    w = torch.randn(tokens, k, device="cuda")
    assert comp.token_order_workspace(comp.FLOAT32 if kind == "float32" else comp.BFLOAT16, tokens, k, hidden) == 8 * tokens * k
    none = torch.zeros(1, dtype=torch.int64, device="cuda")
    outs = [(torch.full((rows, hidden), 3.0, device="cuda", dtype=t), torch.full((rows, hidden), 3.0, device="cuda", dtype=t), torch.zeros(tokens, k, device="cuda"))
            for _ in range(2)]
    for (out, gy, gw), ws, name in zip(outs, (None, none), ("ordered_kernel", "_kernel")):
        comp.token_dispatch(x, pos, counts, offsets, out, workspace=ws)
        assert comp.last_kernel().endswith(name)
        comp.token_combine_backward(x, out, pos, w, counts, offsets, gy, gw, workspace=ws)
        assert comp.last_kernel().endswith(name)
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    some = pos >= 0
    for j in range(k):
        at = pos[:, j].long().clamp(min=0)
        for t0 in range(0, tokens, 16384):
            part = slice(t0, t0 + 16384)
            sums = (x[part].double() * outs[0][0][at[part]].double()).abs().sum(1) * some[part, j]
            assert ((outs[0][2][part, j] - outs[1][2][part, j]).abs().double() <= 2 * hidden * U32 * sums).all()
    if k == 1:                                                         # one product, rounded to fp32 and to the type
        back = torch.zeros(tokens, hidden, device="cuda", dtype=t)
        comp.token_combine(outs[0][0], pos, w, back)
        for t0 in range(0, tokens, 16384):
            part = slice(t0, t0 + 16384)
            want = (w[part] * x[part].float()).to(t) * some[part]
            assert torch.equal(back[part], want)


def test_what_is_not_finite_stays_where_it_is(comp):
    """A NaN or an infinity in a row reaches the tokens of that row alone; rows that no token has are never read into a sum, and
    neither is the padding."""
    import torch
    pos = torch.tensor([[0, 1], [2, -1], [-1, -1]], dtype=torch.int32, device="cuda")
    y = torch.ones(5, 33, device="cuda", dtype=torch.bfloat16)
    y[1], y[3], y[4] = float("inf"), float("nan"), float("nan")
    w = torch.tensor([[1.0, -1.0], [2.0, float("nan")], [float("nan"), float("inf")]], device="cuda")
    out = torch.zeros(3, 33, device="cuda", dtype=torch.bfloat16)
    comp.token_combine(y, pos, w, out)
    assert (out[0] == -float("inf")).all() and (out[1] == 2).all() and (out[2] == 0).all()
    g = torch.ones(3, 33, device="cuda", dtype=torch.bfloat16)
    gy, gw = torch.zeros_like(y), torch.zeros(3, 2, device="cuda")
    counts, offsets = torch.tensor([3], dtype=torch.int32, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    gy.fill_(5)
    comp.token_combine_backward(g, y, pos, w, counts, offsets, gy, gw)
    assert gw.tolist() == [[33, float("inf")], [33, 0], [0, 0]]
    assert gy[:, 0].tolist() == [1, -1, 2, 0, 5]


def test_gradients_against_differences(comp):
    """Combine and dispatch are linear in the rows, the weights and the tokens, so a difference quotient over +-1/2 is exact but
    for roundings.  In units of 2^-24: an output is a sum of two products of |w| <= 1.5 and |y| <= 1.5, one of them moved, so off
    by at most 2 (1.5 + 1) = 5; two losses of 32 outputs times |g| <= 1: 320; the moved value's own rounding, twice, times at
    most 8 products: 16; the gradient of a weight, 8 terms: 64.  In all 400."""
    import torch
    rng = np.random.default_rng(5)
    tokens, k, experts, hidden = 4, 2, 3, 8
    ids = make_ids(rng, tokens, k, experts)
    pos, counts, offsets = sort(comp, ids, experts, 4)
    rows = comp.token_rows(tokens, k, experts, 4)
    x, y, g = (torch.from_numpy(rng.uniform(-1, 1, (n, hidden)).astype(np.float32)).cuda() for n in (tokens, rows, tokens))
    w, gr = torch.from_numpy(rng.uniform(-1, 1, (tokens, k)).astype(np.float32)).cuda(), torch.from_numpy(rng.uniform(-1, 1, (rows, hidden)).astype(np.float32)).cuda()
    gr[int(offsets[-1]):] = 0
    tol = 400 * U32

    def loss(y_, w_):
        out = torch.zeros(tokens, hidden, device="cuda")
        comp.token_combine(y_, pos, w_, out)
        return float((out.double() * g.double()).sum())

    def sent(x_):
        out = torch.zeros(rows, hidden, device="cuda")
        comp.token_dispatch(x_, pos, counts, offsets, out)
        return float((out.double() * gr.double()).sum())
    gy, gw, gx = torch.zeros_like(y), torch.zeros_like(w), torch.zeros_like(x)
    comp.token_combine_backward(g, y, pos, w, counts, offsets, gy, gw)
    comp.token_dispatch_backward(gr, pos, gx)
    for of, grad, f in ((y, gy, lambda v: loss(v, w)), (w, gw, lambda v: loss(y, v)), (x, gx, sent)):
        for i in range(0, of.numel(), 3):
            up, down = of.clone(), of.clone()
            up.view(-1)[i] += 0.5
            down.view(-1)[i] -= 0.5
            assert abs(f(up) - f(down) - float(grad.view(-1)[i])) <= tol


def test_refusals_of_the_binding(comp):
    import torch
    pos = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    counts, offsets = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 8, device="cuda")
    for call in (lambda: comp.token_dispatch(x, pos, counts, offsets, torch.zeros(4, 7, device="cuda")),
                 lambda: comp.token_dispatch(x, pos, counts, offsets, torch.zeros(4, 8, device="cuda", dtype=torch.float16)),
                 lambda: comp.token_dispatch(x, pos, counts, offsets, torch.zeros(4, 8)),
                 lambda: comp.token_dispatch(x, pos, counts, offsets[:3], torch.zeros(4, 8, device="cuda")),
                 lambda: comp.token_dispatch(x, pos[:1], counts, offsets, torch.zeros(4, 8, device="cuda")),
                 lambda: comp.token_dispatch(x, pos.long(), counts, offsets, torch.zeros(4, 8, device="cuda")),
                 lambda: comp.token_combine(x.t(), pos, None, torch.zeros(2, 2, device="cuda")),
                 lambda: comp.token_combine(x.double(), pos, None, torch.zeros(2, 8, device="cuda").double()),
                 lambda: comp.token_combine(x, pos, torch.zeros(2, 3, device="cuda"), torch.zeros(2, 8, device="cuda")),
                 lambda: comp.token_combine(x, pos, torch.zeros(2, 2, device="cuda").t(), torch.zeros(2, 8, device="cuda").double()),
                 lambda: comp.token_combine(x, pos, torch.zeros(3, device="cuda"), torch.zeros(2, 8, device="cuda")),
                 lambda: comp.token_combine_backward(x, None, pos, None, counts, offsets, torch.zeros(4, 8, device="cuda"), torch.zeros(2, 2, device="cuda")),
                 lambda: comp.token_combine_backward(x, torch.zeros(3, 8, device="cuda"), pos, None, counts, offsets, torch.zeros(4, 8, device="cuda")),
                 lambda: comp.token_sort(pos, 3, pos.view(4, 1), counts, offsets),
                 lambda: comp.token_sort(pos.float(), 3, pos, counts, offsets),
                 lambda: comp.token_combine(torch.zeros(1, 8, device="cuda").expand(3, 8), pos, None, torch.zeros(2, 8, device="cuda"))):
        with pytest.raises((ValueError, comp.CclError)):
            call()


def test_rows_past_32_bits_of_bytes(comp):
    """270,001 rows of 16 KiB: copies and products by one, to the bit, in both forms."""
    import torch
    tokens, hidden, experts = 270001, 8192, 4
    rng = np.random.default_rng(3)
    pos, counts, offsets = sort(comp, make_ids(rng, tokens, 1, experts), experts, 16)
    rows = comp.token_rows(tokens, 1, experts, 16)
    x = torch.randn(1, hidden, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16().repeat(tokens, 1)
    x[:, 0] = torch.arange(tokens, device="cuda").bfloat16()
    x[:, 1] = (torch.arange(tokens, device="cuda") % 251).bfloat16()
    x[:, hidden - 1] = (torch.arange(tokens, device="cuda") % 241).bfloat16()
    none = torch.zeros(1, dtype=torch.int64, device="cuda")
    out, back = torch.empty(rows, hidden, device="cuda", dtype=torch.bfloat16), torch.empty_like(x)
    ones = torch.ones(tokens, 1, device="cuda")
    assert out.numel() * 2 > 1 << 32
    for ws in (None, none):
        for call in (lambda: comp.token_dispatch(x, pos, counts, offsets, out, workspace=ws),
                     lambda: comp.token_combine_backward(x, None, pos, ones, counts, offsets, out, workspace=ws)):
            out.fill_(3.0)
            call()
            back.zero_()
            comp.token_combine(out, pos, ones, back)
            for t0 in range(0, tokens, 1 << 15):
                part = slice(t0, t0 + (1 << 15))
                assert torch.equal(out[pos[part, 0].long()], x[part]) and torch.equal(back[part], x[part])
            end, begin = int(offsets[-1]), offsets[:-1] + counts
            for e in range(experts):
                assert not out[int(begin[e]):int(offsets[e + 1])].any()
            assert (out[end:] == 3).all()
