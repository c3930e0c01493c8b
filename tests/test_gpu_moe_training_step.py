"""The operators together, as one training step of an expert-parallel layer on one rank uses them: tokens sorted by expert and
dispatched, the experts' products, the weighted sum, both gradients, the reduce of the weight gradients over the peers in one
fusion buffer, the norm with its clip coefficient and the AdamW step from that buffer -- against the same step in 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TOKENS, TOP_K, EXPERTS, HIDDEN, ALIGN, PEERS = 37, 2, 5, 24, 4, 3


@pytest.fixture(scope="module")
def comp():
    import torch
    assert torch.cuda.is_available(), "needs a GPU"
    import oneccl_amd.comp as c
    c.lib()
    return c


class Step:
    """Buffers and weights of a rank, all float32, and the step over them; nothing is allocated in run()."""

    def __init__(self, comp, seed, eight=False):
        import torch
        rng = np.random.default_rng(seed)
        self.comp = comp

        def dev(*shape, scale=1.0):
            return torch.from_numpy((scale * rng.standard_normal(shape)).astype(np.float32)).cuda()
        ids = np.argsort(rng.standard_normal((TOKENS, EXPERTS)), axis=1)[:, :TOP_K].astype(np.int64)
        ids[5] = -1                                                        # a masked token
        ids[ids == 3] = 2                                                  # expert 3 has nothing to do; some tokens name 2 twice
        self.ids = torch.from_numpy(ids).cuda()
        self.x, self.gate, self.target = dev(TOKENS, HIDDEN), dev(TOKENS, TOP_K, scale=0.5), dev(TOKENS, HIDDEN)
        # one weight per expert, a shared scale behind the sum
        self.params = [dev(HIDDEN, HIDDEN, scale=HIDDEN ** -0.5) for _ in range(EXPERTS)] + [dev(HIDDEN)]
        counts = [p.numel() for p in self.params]
        self.plan = comp.FusionPlan(counts, comp.FLOAT32, 1024)
        n = self.plan.elements
        self.first = [self.plan.offset(i) // 4 for i in range(len(counts))]
        self.peers = [dev(n, scale=0.3) for _ in range(PEERS)]             # what the other ranks sent
        rows = comp.token_rows(TOKENS, TOP_K, EXPERTS, ALIGN)
        self.pos = torch.zeros(TOKENS, TOP_K, dtype=torch.int32, device="cuda")
        self.counts, self.offsets = torch.zeros(EXPERTS, dtype=torch.int32, device="cuda"), torch.zeros(EXPERTS + 1, dtype=torch.int32, device="cuda")
        self.rows, self.act, self.g_act, self.g_rows = (torch.zeros(rows, HIDDEN, device="cuda") for _ in range(4))
        self.out, self.y, self.g_out, self.g_x = (torch.zeros(TOKENS, HIDDEN, device="cuda") for _ in range(4))
        self.g_gate = torch.zeros(TOKENS, TOP_K, device="cuda")
        self.grads = [torch.zeros_like(p) for p in self.params]
        self.reduced = torch.zeros(n, device="cuda")
        self.packed = torch.zeros(n, device="cuda")
        if eight:
            self.m, self.v = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
            self.scales = torch.zeros(2 * -(-n // 256), dtype=torch.uint8, device="cuda")
        else:
            self.m, self.v, self.scales = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), None
        self.result = torch.zeros(2, device="cuda")
        self.norm_ws = torch.zeros(self.plan.norm_workspace, dtype=torch.uint8, device="cuda")
        self.step, self.lr = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.full((1,), 1e-2, device="cuda")
        # row r belongs to expert e: a mask in place of host-side segment sizes (the sizes stay on the device)
        self.row = torch.arange(rows, device="cuda")[:, None]
        self.max_norm, self.hyper = 0.5, dict(beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)

    def run(self):
        import torch
        c = self.comp
        c.token_sort(self.ids, EXPERTS, self.pos, self.counts, self.offsets, align=ALIGN)
        c.token_dispatch(self.x, self.pos, self.counts, self.offsets, self.rows)
        self.act.zero_()
        masks = [((self.row >= self.offsets[e]) & (self.row < self.offsets[e + 1])).float() for e in range(EXPERTS)]
        for e in range(EXPERTS):
            self.act += masks[e] * (self.rows @ self.params[e])
        c.token_combine(self.act, self.pos, self.gate, self.out)
        torch.mul(self.out, self.params[-1], out=self.y)
        # loss = sum (y - target)^2 / 2
        g_y = self.y - self.target
        self.grads[-1].copy_((g_y * self.out).sum(0))
        torch.mul(g_y, self.params[-1], out=self.g_out)
        c.token_combine_backward(self.g_out, self.act, self.pos, self.gate, self.counts, self.offsets, self.g_act, self.g_gate)
        self.g_rows.zero_()
        for e in range(EXPERTS):
            self.grads[e].copy_((self.rows * masks[e]).t() @ self.g_act)
            self.g_rows += masks[e] * (self.g_act @ self.params[e].t())
        c.token_dispatch_backward(self.g_rows, self.pos, self.g_x)
        self.plan.pack(self.grads, self.packed)
        c.comp_reduce_n(c.FLOAT32, c.SUM, [self.packed] + self.peers, self.reduced, self.reduced.numel())
        self.step += 1
        self.plan.norm(self.reduced, self.result, multiplier=1 / (PEERS + 1), max_norm=self.max_norm, workspace=self.norm_ws)
        self.plan.adamw(self.params, self.reduced, self.m, self.v, lr=0.0, scales=self.scales, grad_scale=self.result[1:], step_ptr=self.step,
                        lr_ptr=self.lr, **self.hyper)

    def state(self):
        return [p.clone() for p in self.params] + [t.clone() for t in (self.m, self.v, self.y, self.g_x, self.g_gate, self.result)]


def reference(s):
    """One step in 64 bits with torch's own gradients (the first: states zero, t = 1): weights before and after, g_x, g_gate, norm."""
    import torch
    ids = s.ids.cpu()
    x, gate = s.x.cpu().double().requires_grad_(), s.gate.cpu().double().requires_grad_()
    ws = [p.cpu().double().requires_grad_() for p in s.params]
    rows = []
    for t in range(TOKENS):
        acc = torch.zeros(HIDDEN, dtype=torch.float64)
        for j in range(TOP_K):
            if 0 <= ids[t, j] < EXPERTS:
                acc = acc + gate[t, j] * (x[t] @ ws[int(ids[t, j])])
        rows.append(acc)
    y = torch.stack(rows) * ws[-1]
    ((y - s.target.cpu().double()) ** 2 / 2).sum().backward()
    peers = [sum(p[f:f + w.numel()].cpu().double().reshape(w.shape) for p in s.peers) for f, w in zip(s.first, ws)]
    grads = [(w.grad if w.grad is not None else torch.zeros_like(w)) + p for w, p in zip(ws, peers)]
    norm = math.sqrt(sum(float((g ** 2).sum()) for g in grads)) / (PEERS + 1)
    coef = min(1.0, s.max_norm / (norm + 1e-6)) / (PEERS + 1)
    after = []
    for w, g in zip(ws, grads):
        g = g * coef
        m, v = 0.1 * g, 0.05 * g * g
        after.append(w.detach() * (1 - 1e-2 * 0.1) - 1e-2 * (m / 0.1) / (torch.sqrt(v / 0.05) + 1e-8))
    return y.detach(), x.grad, gate.grad, norm, grads, after


def magnitudes(s):
    """What the step's outputs would be if nothing in it cancelled: every sum over the absolute values of its terms."""
    import torch
    ids = s.ids.cpu()
    x, gate, target = (t.cpu().double().abs() for t in (s.x, s.gate, s.target))
    ws = [p.cpu().double().abs() for p in s.params]
    act = [[x[t] @ ws[int(e)] if 0 <= e < EXPERTS else torch.zeros(HIDDEN, dtype=torch.float64) for e in ids[t]] for t in range(TOKENS)]
    out = torch.stack([sum(gate[t, j] * act[t][j] for j in range(TOP_K)) for t in range(TOKENS)])
    y = out * ws[-1]
    g_y = y + target
    g_out = g_y * ws[-1]
    g_x, g_gate, grads = torch.zeros_like(x), torch.zeros_like(gate), [torch.zeros_like(w) for w in ws]
    grads[-1] = (g_y * out).sum(0)
    for t in range(TOKENS):
        for j, e in enumerate(ids[t].tolist()):
            if 0 <= e < EXPERTS:
                g_gate[t, j] = (g_out[t] * act[t][j]).sum()
                g_x[t] += gate[t, j] * (ws[e] @ g_out[t])
                grads[e] += torch.outer(x[t], gate[t, j] * g_out[t])
    for f, g in zip(s.first, grads):
        g += sum(p[f:f + g.numel()].cpu().double().abs().reshape(g.shape) for p in s.peers)
    return y, g_x, g_gate, grads


def test_one_step_against_64_bits(comp):
    """No value is behind more than 180 fp32 roundings: 24 of an expert's product, 10 of the masked sum over the experts, 2 of
    combine, 4 of the loss's gradient and the weights, 24 of the second product, at most 98 rows of a weight's gradient, 4 of the
    reduce, and each of them is 2^-24 of a partial sum, which the sum of the absolute values bounds."""
    import torch
    s = Step(comp, 3)
    y, g_x, g_gate, norm, grads, after = reference(s)
    my, mx, mg, mw = magnitudes(s)
    assert s.rows.shape[0] <= 98
    s.run()
    for got, want, most in ((s.y, y, my), (s.g_x, g_x, mx), (s.g_gate, g_gate, mg)):
        assert ((got.cpu().double() - want).abs() <= 180 * U * most).all()
    off = 0.0
    for f, g, most in zip(s.first, grads, mw):
        got = s.reduced[f:f + g.numel()].cpu().double().reshape(g.shape)
        assert ((got - g).abs() <= 180 * U * most).all()
        off += float(((180 * U * most) ** 2).sum())
    assert abs(s.result[0].item() - norm) <= math.sqrt(off) / (PEERS + 1) + 18 * U * norm
    # The first step moves a weight by lr * g / (|g| + eps): where g is sure of its sign (its error under 1/100 of it) and far
    # above eps, that is lr to 1e-5 of it whatever the rest of g; the weight itself takes 3 roundings.
    for p, w, g, most in zip(s.params, after, grads, mw):
        sure = (g.abs() > 18000 * U * most) & (g.abs() > 1e-2)
        assert ((p.cpu().double() - w)[sure].abs() <= 1e-2 * 1e-5 + 15 * U * 1e-2 + 3 * U * w[sure].abs()).all()
        assert sure.any()


@pytest.mark.parametrize("eight", [False, True])
def test_the_step_captured_and_replayed(comp, eight):
    """Five steps of one graph against five eager steps, bit for bit, with eager work and synchronizations between the replays; an
    eager step object lives on meanwhile."""
    import torch
    eager, graphed = Step(comp, 8, eight), Step(comp, 8, eight)
    warm = Step(comp, 9, eight)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm.run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        graphed.run()
    for rep in range(5):
        eager.run()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        warm.run()                              # other eager work, other buffers
        for a, b in zip(eager.state(), graphed.state()):
            assert torch.equal(a, b), rep


def test_two_streams_at_once(comp):
    """Two steps on two streams, of default priority, at once: as if alone."""
    import torch
    alone = [Step(comp, 20 + i) for i in range(2)]
    both = [Step(comp, 20 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s in alone:
            s.run()
            torch.cuda.synchronize()
        for s, st in zip(both, streams):
            with torch.cuda.stream(st):
                s.run()
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        for x, y in zip(a.state(), b.state()):
            assert torch.equal(x, y)


def test_a_stream_that_is_not_the_current_one(comp):
    """stream= names the stream of the call: work before it on that stream is seen, the current stream need not be waited for."""
    import torch
    st = torch.cuda.Stream()
    x = torch.zeros(4, 8, device="cuda")
    pos = torch.tensor([[0], [1], [2], [3]], dtype=torch.int32, device="cuda")
    counts, offsets = torch.tensor([4], dtype=torch.int32, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    out = torch.zeros(4, 8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        x.fill_(3.0)
    comp.token_dispatch(x, pos, counts, offsets, out, stream=st)
    st.synchronize()
    assert (out == 3).all()


@pytest.mark.parametrize("variant", [0, 8])
def test_scratch_memory_that_the_binding_allocates_in_a_graph_and_on_a_side_stream(comp, variant):
    """Sort, dispatch, gradients and norm with their scratch memory from the call itself: captured (the graph's own pool keeps it),
    replayed between eager work, and on a stream that is not the current one while the current one allocates and writes."""
    import torch
    rng = np.random.default_rng(4)
    tokens, k, experts, hidden = 9001, 2, 33, 40                       # more entries than one block sorts
    ids = torch.from_numpy(rng.integers(-1, experts, (tokens, k)).astype(np.int32)).cuda()
    x, w = torch.randn(tokens, hidden, device="cuda").bfloat16(), torch.rand(tokens, k, device="cuda")
    rows = comp.token_rows(tokens, k, experts, 8)
    plan = comp.FusionPlan([100000, 77777], comp.FLOAT32, 1)
    grads = torch.randn(plan.elements, device="cuda")

    def buffers():
        return dict(pos=torch.zeros(tokens, k, dtype=torch.int32, device="cuda"), counts=torch.zeros(experts, dtype=torch.int32, device="cuda"),
                    offsets=torch.zeros(experts + 1, dtype=torch.int32, device="cuda"), out=torch.zeros(rows, hidden, device="cuda").bfloat16(),
                    gy=torch.zeros(rows, hidden, device="cuda").bfloat16(), gw=torch.zeros(tokens, k, device="cuda"), res=torch.zeros(2, device="cuda"))

    def run(b, stream=None):
        comp.token_sort(ids, experts, b["pos"], b["counts"], b["offsets"], align=8, stream=stream)
        comp.token_dispatch(x, b["pos"], b["counts"], b["offsets"], b["out"], stream=stream)
        comp.token_combine_backward(x, b["out"], b["pos"], w, b["counts"], b["offsets"], b["gy"], b["gw"], stream=stream)
        plan.norm(grads, b["res"], max_norm=1.0, stream=stream)
    comp.set_param("variant", variant)
    try:
        want, got = buffers(), buffers()
        run(want)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(got)
        for rep in range(4):
            for t in got.values():
                t.zero_()
            junk = [torch.full((1 << 18,), 7, device="cuda", dtype=torch.int32) for _ in range(4)]
            run(buffers())
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(want[n], got[n]) for n in want), rep
        for side in (torch.cuda.Stream(), torch.cuda.Stream().cuda_stream):
            got = buffers()
            torch.cuda.synchronize()
            for _ in range(3):
                run(got, stream=side)
                junk = [torch.full((1 << 18,), 7, device="cuda", dtype=torch.int32) for _ in range(8)]
            torch.cuda.synchronize()
            assert all(torch.equal(want[n], got[n]) for n in want)
    finally:
        comp.set_param("variant", 0)
