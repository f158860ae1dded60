"""Routing (frc_route_device, frc_balance_device, frc_route_backward_device) against float64.

Expert ids and counts are equal.  Tolerances, u = 2^-24 (half an fp32 step), R = the largest max - l of a row that
still counts (exp(-104) is below every fp32 number):
  gates:  exp's argument is one fp32 difference (R u relative in the result) and exp itself 2 steps (4 u); the sum of
          ten positive terms and the quotient 12 u; twice the first two for numerator and sum: (2 R + 20) u relative.
  p:      the argument is rounded twice (2 R u), exp2 2 steps (4 u); E positive terms in a tree 10 u, the quotient
          3 u: (4 R + 32) u relative; prob and loss sum up to T of them one by one: + T u.
  gradients: the balance term is scale p_e (count_e - dot): with the size s = scale p_e (count_e + dot) off by
          (8 R + 600) u s (dot sums E products, 512 u); the routing term g (d - sum g d) by (4 R + 60) u g (|d| + sum g |d|);
          a bf16 result adds 2^-8 of the value.
Everything below 2^-126 may be flushed."""
import numpy as np
import pytest

import fronk_b200 as fb

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TINY = 2.0 ** -126


@pytest.fixture(scope="module")
def ctx(gpu):
    with fb.Context(0, 512) as c:
        yield c


class Reference:
    """Float64 routing of logits [T][E] (-inf masked), valid [T] bools, shared logits [T] or None."""

    def __init__(self, l, valid=None, shared=None, expert=None):
        T, E = l.shape
        self.E, self.T = E, T
        self.valid = np.ones(T, bool) if valid is None else valid
        l = np.where(self.valid[:, None], l, -np.inf).astype(np.float64)
        self.l = l
        if expert is None:
            expert = np.argsort(-l, axis=1, kind="stable")[:, :10]
            expert[~self.valid] = np.arange(10)
        self.expert = expert
        self.p, self.R = self.softmax(l)
        self.le = np.take_along_axis(l, expert, 1)
        self.g, self.Rg = self.softmax(self.le)
        self.gs = np.zeros(T)
        if shared is not None:
            with np.errstate(over="ignore"):
                self.gs = np.where(self.valid, 1 / (1 + np.exp(-np.where(self.valid, shared, 0.0))), 0)
        taken = self.valid[:, None] & ~np.isneginf(self.le)
        self.n = int(self.valid.sum())
        self.count = np.append(np.bincount(expert[taken], minlength=E), self.n)
        self.prob = self.p.sum(0) / max(self.n, 1)
        self.loss = E * float(self.count[:E] @ self.prob) / (10 * max(self.n, 1))

    @staticmethod
    def softmax(l):
        m = l.max(1, keepdims=True)
        m = np.where(np.isneginf(m), 0, m)
        z = np.exp(l - m)
        s = z.sum(1, keepdims=True)
        fin = np.where(np.isneginf(l), m, l)
        return np.divide(z, s, out=np.zeros_like(z), where=s > 0), np.minimum((m - fin).max(1, keepdims=True), 104)

    def backward(self, d_gate=None, d_loss=None, shared=False):
        """(gradient, its tolerance) of the columns [E (+ 1)]."""
        E, T = self.E, self.T
        d = np.zeros((T, E + int(shared)))
        tol = np.full_like(d, TINY)
        if d_loss is not None and self.n:
            c = self.count[:E].astype(np.float64)
            dot = (self.p @ c)[:, None]
            scale = d_loss * E / (10 * float(self.n) ** 2)
            d[:, :E] += scale * self.p * (c - dot)
            tol[:, :E] += (8 * self.R + 600) * U * np.abs(scale) * self.p * (c + dot)
        if d_gate is not None:
            dg = d_gate[:, :10]
            row = np.arange(T)[:, None]
            np.add.at(d, (row, self.expert), self.g * (dg - (self.g * dg).sum(1, keepdims=True)))
            size = self.g * (np.abs(dg) + (self.g * np.abs(dg)).sum(1, keepdims=True))
            np.add.at(tol, (row, self.expert), (4 * self.Rg + 60) * U * size)
            if shared:
                d[:, E] = np.where(self.valid, self.gs * (1 - self.gs) * d_gate[:, 10], 0)
                # s (1 - s) from an fp32 s: 1 - s loses what s rounds away, 4 u of s
                tol[:, E] += (8 * self.gs * U + 60 * U * self.gs * (1 - self.gs)) * np.abs(d_gate[:, 10])
        return d, tol


class Buffers:
    """Device buffers of one call; rows `pad` elements apart, behind an odd first element."""

    def __init__(self, l, dtype=fb.F32, pad=0, valid=None, shared=None, offset=0):
        import torch
        self.dtype, self.flags = dtype, fb.ROUTE_SHARED if shared is not None else 0
        T, self.E = l.shape
        self.T, self.cols = T, self.E + int(shared is not None)
        self.stride = self.cols + pad
        full = np.full((T, self.stride), np.nan, np.float32)
        full[:, :self.E] = l
        if shared is not None:
            full[:, self.E] = shared
        td = torch.bfloat16 if dtype == fb.BF16 else torch.float32
        store = torch.zeros(offset + T * self.stride, dtype=td, device="cuda")
        self.logits = store[offset:].view(T, self.stride)
        self.logits.copy_(torch.from_numpy(full))
        self.valid = None if valid is None else torch.from_numpy(valid.astype(np.uint8)).cuda()
        self.expert = torch.full((T, 10), -1, dtype=torch.int16, device="cuda")
        self.gate = torch.full((T, 11), float("nan"), device="cuda")
        self.loss = torch.full((1,), float("nan"), device="cuda")
        self.count = torch.full((self.E + 1,), -1, dtype=torch.int32, device="cuda")
        self.prob = torch.full((self.E,), float("nan"), device="cuda")
        ws = fb.balance_workspace(T, self.E)
        self.ws = torch.randint(0, 256, (ws,), dtype=torch.uint8, device="cuda")
        self.balance = fb.Balance(self.loss.data_ptr(), self.count.data_ptr(), self.prob.data_ptr(),
                                  self.ws.data_ptr(), ws)

    def _valid(self):
        return None if self.valid is None else self.valid.data_ptr()

    def seen(self):
        """What the device sees of the logits and shared logits, float64."""
        v = self.logits.float().cpu().numpy().astype(np.float64)
        return v[:, :self.E], (v[:, self.E] if self.flags else None)

    def route(self, ctx, balance=False, stream=None):
        import torch
        s = torch.cuda.current_stream().cuda_stream if stream is None else stream
        ctx.route_device(self.T, self.E, self.logits.data_ptr(), self.expert.data_ptr(), self.gate.data_ptr(),
                         self.stride, self.dtype, self._valid(), self.flags, self.balance if balance else None, s)

    def stats(self, ctx, expert, stream=None):
        import torch
        s = torch.cuda.current_stream().cuda_stream if stream is None else stream
        ctx.balance_device(self.T, self.E, self.logits.data_ptr(), expert.data_ptr(), self.balance, self.stride,
                           self.dtype, self._valid(), s)

    def backward(self, ctx, out, expert, d_gate, d_loss, stream=None):
        import torch
        s = torch.cuda.current_stream().cuda_stream if stream is None else stream
        ctx.route_backward_device(
            self.T, self.E, self.logits.data_ptr(), None if expert is None else expert.data_ptr(), out.data_ptr(),
            None if d_gate is None else d_gate.data_ptr(), None if d_loss is None else self.count.data_ptr(),
            None if d_loss is None else d_loss.data_ptr(), self.stride, out.shape[1], self.dtype, self._valid(),
            self.flags, s)


def check_route(b, ref):
    assert np.array_equal(b.expert.cpu().numpy().astype(np.int64), ref.expert)
    g = b.gate.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(g[:, :10] - ref.g) <= (2 * ref.Rg + 20) * U * ref.g + TINY)
    assert np.all(np.abs(g[:, 10] - ref.gs) <= 16 * U * ref.gs + TINY)


def check_stats(b, ref):
    assert np.array_equal(b.count.cpu().numpy(), ref.count)
    rel = (4 * (ref.R[ref.valid].max() if ref.n else 0) + 32 + b.T) * U
    prob = b.prob.cpu().numpy().astype(np.float64)
    assert np.all(np.abs(prob - ref.prob) <= rel * ref.prob + TINY)
    assert abs(float(b.loss[0]) - ref.loss) <= (rel + 4 * U) * ref.loss


def logits_of(kind, T, E, rng):
    l = rng.standard_normal((T, E)) * 2
    if kind == "ties":
        l = np.round(l)
    elif kind == "equal":
        l[:] = 0.25
    elif kind == "zeros":
        l = np.where(rng.random((T, E)) < 0.5, 0.0, -0.0)  # +0 and -0 are equal
    elif kind == "masked":
        l[rng.random((T, E)) < 0.5] = -np.inf
    elif kind == "few":  # fewer than ten left, in some rows one or none
        keep = rng.integers(0, 9, T)
        for t in range(T):
            m = rng.permutation(E)[keep[t]:]
            l[t, m] = -np.inf
    elif kind == "lowest":  # masks of the type's lowest value are numbers
        l[rng.random((T, E)) < 0.9] = -3e38
        l[0] = -3e38
    elif kind == "wide":
        l *= 40
    elif kind == "sorted":
        l = np.sort(l, 1) if rng.random() < 0.5 else -np.sort(-l, 1)
    elif kind == "large":
        l = l * 1e37
    elif kind == "largest zeros":  # a dozen of +0 and -0 above the rest
        l = -np.abs(l) - 0.1
        for t in range(T):
            l[t, rng.permutation(E)[:13]] = 0.0
        l = np.where((l == 0) & (rng.random((T, E)) < 0.5), -0.0, l)
    return l


KINDS = ["normal", "ties", "equal", "zeros", "masked", "few", "lowest", "wide", "sorted", "large", "largest zeros"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,E", [(1, 10), (1, 512), (2, 511), (7, 33), (64, 512), (129, 160), (1000, 257), (40, 32)])
@pytest.mark.parametrize("dtype", [fb.F32, fb.BF16])
def test_route_and_balance(ctx, kind, T, E, dtype):
    rng = np.random.default_rng(KINDS.index(kind) * 7919 + T * 31 + E)
    for variant in range(3):
        shared = rng.standard_normal(T) * 4 if variant else None
        valid = rng.random(T) < 0.7 if variant == 2 else None
        b = Buffers(logits_of(kind, T, E, rng), dtype, pad=(0, 5, 7)[variant], valid=valid, shared=shared,
                    offset=(0, 1, 8)[variant])
        l, sh = b.seen()
        ref = Reference(l, valid, sh)
        b.route(ctx)
        assert ctx.status() == fb.OK
        check_route(b, ref)
        b.expert.fill_(-1)
        b.gate.fill_(float("nan"))
        b.route(ctx, balance=True)
        assert ctx.status() == fb.OK
        check_route(b, ref)
        check_stats(b, ref)
        first = (b.loss.clone(), b.prob.clone())
        b.loss.fill_(-1)
        b.prob.fill_(-1)
        b.count.fill_(-1)
        b.stats(ctx, b.expert)
        assert ctx.status() == fb.OK
        check_stats(b, ref)
        b.route(ctx, balance=True)
        assert ctx.status() == fb.OK and float(b.loss) == float(first[0]) and bool((b.prob == first[1]).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,E", [(1, 10), (3, 512), (65, 200), (500, 511)])
@pytest.mark.parametrize("dtype", [fb.F32, fb.BF16])
def test_backward(ctx, kind, T, E, dtype):
    import torch
    rng = np.random.default_rng(KINDS.index(kind) * 104729 + T * 31 + E)
    for variant in range(3):
        shared = rng.standard_normal(T) * 4 if variant else None
        valid = rng.random(T) < 0.7 if variant == 2 else None
        b = Buffers(logits_of(kind, T, E, rng), dtype, pad=(0, 5, 7)[variant], valid=valid, shared=shared,
                    offset=(0, 1, 8)[variant])
        l, sh = b.seen()
        ref = Reference(l, valid, sh)
        b.route(ctx, balance=True)
        dg = rng.standard_normal((T, 11)).astype(np.float32)
        d_gate = torch.from_numpy(dg).cuda()
        d_loss = torch.full((1,), -0.75, device="cuda")
        for use_gate, use_loss in [(True, True), (True, False), (False, True)]:
            out = torch.full((T, b.cols + 3), 5.0, dtype=b.logits.dtype, device="cuda")
            b.backward(ctx, out, b.expert if use_gate else None, d_gate if use_gate else None,
                       d_loss if use_loss else None)
            assert ctx.status() == fb.OK
            d, tol = ref.backward(dg.astype(np.float64) if use_gate else None, -0.75 if use_loss else None,
                                  shared is not None)
            got = out.float().cpu().numpy().astype(np.float64)
            tol = tol + (2.0 ** -8 * np.abs(d) + 2.0 ** -133 if dtype == fb.BF16 else 0)
            assert np.all(np.abs(got[:, :b.cols] - d) <= tol), (np.abs(got[:, :b.cols] - d) / tol).max()
            assert np.all(got[:, b.cols:] == 5)
        # in place
        keep = b.logits.clone()
        out = torch.zeros(T, b.stride, dtype=b.logits.dtype, device="cuda")
        b.backward(ctx, out, b.expert, d_gate, d_loss)
        b.backward(ctx, b.logits, b.expert, d_gate, d_loss)
        assert ctx.status() == fb.OK
        assert torch.equal(b.logits[:, :b.cols], out[:, :b.cols])
        assert torch.equal(torch.isnan(b.logits[:, b.cols:]), torch.isnan(keep[:, b.cols:]))


def test_gradient_against_differences(ctx):
    """The gradient of sum(c gate) + 0.5 loss(prob) by central differences of the float64 formulas (the chosen set and
    the counts held)."""
    import torch
    rng = np.random.default_rng(9)
    T, E = 6, 24
    b = Buffers(rng.standard_normal((T, E)), shared=rng.standard_normal(T))
    l, sh = b.seen()
    ref = Reference(l, None, sh)
    b.route(ctx, balance=True)
    c = rng.standard_normal((T, 11))
    out = torch.zeros(T, b.cols, device="cuda")
    b.backward(ctx, out, b.expert, torch.from_numpy(c.astype(np.float32)).cuda(), torch.full((1,), 0.5, device="cuda"))

    def value(full):
        r = Reference(full[:, :E], None, full[:, E], expert=ref.expert)
        loss = E * float(ref.count[:E] @ r.prob) / (10 * T)
        return float((c[:, :10] * r.g).sum() + (c[:, 10] * r.gs).sum()) + 0.5 * loss

    full = np.concatenate([l, sh[:, None]], 1)
    h = 1e-5
    for t in range(T):
        for e in range(E + 1):
            up, down = full.copy(), full.copy()
            up[t, e] += h
            down[t, e] -= h
            # differences are good to h^2 / 6 third derivatives (below 1e-9 here) and 2^-52 |value| / h
            assert abs((value(up) - value(down)) / (2 * h) - float(out[t, e])) < 1e-6 * (1 + abs(c[t]).max())


@pytest.mark.parametrize("kind", ["normal", "ties", "zeros", "masked", "few", "lowest", "largest zeros"])
@pytest.mark.parametrize("T,E,dtype,pad", [(1301, 300, fb.F32, 0), (1400, 130, fb.F32, 2), (4999, 512, fb.F32, 4),
                                           (5000, 512, fb.BF16, 0), (1300, 261, fb.BF16, 3), (1299, 505, fb.BF16, 7)])
def test_large_calls(ctx, kind, T, E, dtype, pad):
    """Rows that pass through shared memory: aligned ones of many tokens, the last columns partly past E."""
    import torch
    rng = np.random.default_rng(T * 13 + E)
    shared = rng.standard_normal(T) if E in (261, 505) else None
    valid = rng.random(T) < 0.7
    b = Buffers(logits_of(kind, T, E, rng), dtype, pad=pad - (shared is not None), valid=valid, shared=shared)
    assert b.stride * b.logits.element_size() % 16 == 0
    l, sh = b.seen()
    ref = Reference(l, valid, sh)
    b.route(ctx)
    assert ctx.status() == fb.OK
    check_route(b, ref)
    ids = b.expert.clone()
    b.expert.fill_(-1)
    b.gate.fill_(float("nan"))
    b.route(ctx, balance=True)
    assert ctx.status() == fb.OK
    check_route(b, ref)
    check_stats(b, ref)
    assert bool(torch.equal(ids, b.expert))
    b.count.fill_(-1)
    b.prob.fill_(-1)
    b.stats(ctx, ids)
    assert ctx.status() == fb.OK
    check_stats(b, ref)


@pytest.mark.parametrize("T", [160, 161, 168, 169, 512, 513, 520])
@pytest.mark.parametrize("E,dtype", [(512, fb.F32), (37, fb.F32), (300, fb.BF16)])
def test_calls_of_hundreds(ctx, T, E, dtype):
    """Around the sizes where statistics change from one cluster to a CTA for eight rows and a launch behind them."""
    rng = np.random.default_rng(T * 7 + E)
    valid = rng.random(T) < 0.8
    b = Buffers(rng.standard_normal((T, E)) * 2, dtype, valid=valid)
    ref = Reference(b.seen()[0], valid)
    b.route(ctx, balance=True)
    assert ctx.status() == fb.OK
    check_route(b, ref)
    check_stats(b, ref)
    first = (b.loss.clone(), b.prob.clone())
    b.loss.fill_(-1)
    b.count.fill_(-1)
    b.prob.fill_(-1)
    b.stats(ctx, b.expert)
    assert ctx.status() == fb.OK
    check_stats(b, ref)
    b.route(ctx, balance=True)
    assert ctx.status() == fb.OK and float(b.loss) == float(first[0]) and bool((b.prob == first[1]).all())


@pytest.mark.parametrize("E", [512, 100])
def test_many_rows(ctx, E):
    """More rows than the GPU's warps; statistics summed over all of them."""
    rng = np.random.default_rng(E)
    T = 12345
    valid = rng.random(T) < 0.9
    b = Buffers(rng.standard_normal((T, E)) * 2, valid=valid)
    ref = Reference(b.seen()[0], valid)
    b.route(ctx, balance=True)
    assert ctx.status() == fb.OK
    check_route(b, ref)
    check_stats(b, ref)


def test_balance_of_foreign_ids(ctx):
    """Ids chosen elsewhere: not the largest logits, the same id twice, a masked id; ids out of range are reported."""
    import torch
    rng = np.random.default_rng(21)
    T, E = 50, 64
    l = rng.standard_normal((T, E))
    l[:, 3] = -np.inf
    b = Buffers(l)
    ids = rng.integers(0, E, (T, 10))
    ids[:, 1] = ids[:, 0]
    ids[:, 2] = 3
    ref = Reference(b.seen()[0], expert=ids)
    dev = torch.from_numpy(ids.astype(np.int16)).cuda()
    b.stats(ctx, dev)
    assert ctx.status() == fb.OK
    check_stats(b, ref)
    dg = rng.standard_normal((T, 11))
    out = torch.zeros(T, E, device="cuda")
    b.backward(ctx, out, dev, torch.from_numpy(dg.astype(np.float32)).cuda(), torch.ones(1, device="cuda"))
    assert ctx.status() == fb.OK
    d, tol = ref.backward(dg.astype(np.float32).astype(np.float64), 1.0)
    assert np.all(np.abs(out.cpu().numpy() - d) <= tol)
    dev[7, 4] = E
    dev[8, 4] = -1
    b.stats(ctx, dev)
    assert ctx.status() == fb.INVALID
    expect = np.append(np.bincount(np.delete(ids.ravel(), [74, 84])[np.delete(ids.ravel(), [74, 84]) != 3], minlength=E), T)
    assert np.array_equal(b.count.cpu().numpy(), expect)
    b.backward(ctx, out, dev, torch.zeros(T, 11, device="cuda"), None)
    assert ctx.status() == fb.INVALID


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_numeric_rows(ctx, value):
    """A NaN or +inf logit of a valid row is reported and the row is padding; in a padding row it is not looked at."""
    rng = np.random.default_rng(22)
    l = rng.standard_normal((9, 40))
    l[4, 17] = value
    for padding in (False, True):
        valid = np.ones(9, bool)
        valid[4] = not padding
        b = Buffers(l, valid=valid)
        b.route(ctx, balance=True)
        assert ctx.status() == (fb.OK if padding else fb.NUMERIC)
        clean = valid.copy()
        clean[4] = False
        ref = Reference(np.where(np.isfinite(l), b.seen()[0], 0), clean)
        check_route(b, ref)
        check_stats(b, ref)


def test_nothing_valid(ctx):
    import torch
    b = Buffers(np.full((5, 30), np.nan), valid=np.zeros(5, bool))
    b.route(ctx, balance=True)
    out = torch.ones(5, 30, device="cuda")
    b.backward(ctx, out, b.expert, torch.ones(5, 11, device="cuda"), torch.ones(1, device="cuda"))
    assert ctx.status() == fb.OK
    assert float(b.loss) == 0 and not bool(b.count.any()) and not bool(b.prob.any())
    assert not bool(b.gate.any()) and not bool(out.any())
    assert np.array_equal(b.expert.cpu().numpy(), np.tile(np.arange(10), (5, 1)))


def test_refusals(ctx):
    import torch
    b = Buffers(np.zeros((4, 20)))
    out = torch.zeros(4, 20, device="cuda")
    dg, dl = torch.zeros(4, 11, device="cuda"), torch.zeros(1, device="cuda")
    L, e, g, o, n = b.logits.data_ptr(), b.expert.data_ptr(), b.gate.data_ptr(), out.data_ptr(), b.count.data_ptr()
    before = ctx.launches
    short = fb.Balance(b.loss.data_ptr(), n, b.prob.data_ptr(), b.ws.data_ptr(), b.ws.numel() - 1)
    null = fb.Balance(b.loss.data_ptr(), n, None, b.ws.data_ptr(), b.ws.numel())
    odd = fb.Balance(b.loss.data_ptr(), n, b.prob.data_ptr(), b.ws.data_ptr() + 4, b.ws.numel())
    calls = [
        lambda: ctx.route_device(0, 20, L, e, g),
        lambda: ctx.route_device(4, 9, L, e, g, stride=20),
        lambda: ctx.route_device(4, 513, L, e, g, stride=600),
        lambda: ctx.route_device(4, 20, L, e, g, stride=19),
        lambda: ctx.route_device(4, 20, L, e, g, stride=20, flags=fb.ROUTE_SHARED),
        lambda: ctx.route_device(4, 20, L, e, g, type_=2),
        lambda: ctx.route_device(4, 20, None, e, g),
        lambda: ctx.route_device(4, 20, L, None, g),
        lambda: ctx.route_device(4, 20, L, e, None),
        lambda: ctx.route_device(4, 20, L + 2, e, g),
        lambda: ctx.route_device(4, 20, L, e + 1, g),
        lambda: ctx.route_device(4, 20, L, e, g, balance=short),
        lambda: ctx.route_device(4, 20, L, e, g, balance=null),
        lambda: ctx.route_device(4, 20, L, e, g, balance=odd),
        lambda: ctx.balance_device(4, 20, L, None, b.balance),
        lambda: ctx.balance_device(4, 20, L, e, short),
        lambda: ctx.route_backward_device(4, 20, L, e, o),
        lambda: ctx.route_backward_device(4, 20, L, None, o, d_gate_ptr=dg.data_ptr()),
        lambda: ctx.route_backward_device(4, 20, L, e, o, count_ptr=n),
        lambda: ctx.route_backward_device(4, 20, L, e, o, d_loss_ptr=dl.data_ptr()),
        lambda: ctx.route_backward_device(4, 20, L, e, o, d_gate_ptr=dg.data_ptr(), d_stride=19),
        lambda: ctx.route_backward_device(4, 20, L, e, None, d_gate_ptr=dg.data_ptr()),
        lambda: ctx.route_backward_device(4, 20, L, e, L, d_gate_ptr=dg.data_ptr(), d_stride=21),
    ]
    for k, call in enumerate(calls):
        with pytest.raises(fb.FrcError) as err:
            call()
        assert err.value.code == fb.INVALID, k
    assert ctx.launches == before and ctx.status() == fb.OK


def test_offsets_past_32_bits(ctx):
    """More than 2^32 elements between the first and the last row."""
    import torch
    rng = np.random.default_rng(25)
    T, E, stride, last = 1050000, 64, 4100, 40
    logits = torch.zeros(T, stride, dtype=torch.bfloat16, device="cuda")
    assert logits.numel() > 1 << 32
    logits[-last:, :E] = torch.from_numpy(rng.standard_normal((last, E)).astype(np.float32)).cuda()
    expert = torch.full((T, 10), -1, dtype=torch.int16, device="cuda")
    gate = torch.full((T, 11), float("nan"), device="cuda")
    ctx.route_device(T, E, logits.data_ptr(), expert.data_ptr(), gate.data_ptr(), stride=stride, type_=fb.BF16)
    assert ctx.status() == fb.OK
    ref = Reference(logits[-last:, :E].float().cpu().numpy().astype(np.float64))
    assert np.array_equal(expert[-last:].cpu().numpy().astype(np.int64), ref.expert)
    assert bool((expert[:-last] == torch.arange(10, device="cuda", dtype=torch.int16)).all())
    assert np.all(np.abs(gate[-last:, :10].cpu().numpy() - ref.g) <= (2 * ref.Rg + 20) * U * ref.g + TINY)
    dg = torch.zeros(T, 11, device="cuda")
    d = rng.standard_normal((last, 11)).astype(np.float32)
    dg[-last:] = torch.from_numpy(d).cuda()
    ctx.route_backward_device(T, E, logits.data_ptr(), expert.data_ptr(), logits.data_ptr(), d_gate_ptr=dg.data_ptr(),
                              stride=stride, d_stride=stride, type_=fb.BF16)
    assert ctx.status() == fb.OK
    want, tol = ref.backward(d.astype(np.float64))
    got = logits[-last:, :E].float().cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got - want) <= tol + 2.0 ** -8 * np.abs(want) + 2.0 ** -133)
    assert not bool(logits[:-last].any())


@pytest.mark.parametrize("T", [300, 2000])
def test_graphs_and_streams(ctx, T):
    """Two captured graphs with workspaces of their own, replayed side by side on new logits."""
    import torch
    rng = np.random.default_rng(23)
    E = 512
    bs = [Buffers(np.zeros((T, E))) for _ in range(2)]
    outs = [torch.zeros(T, E, device="cuda") for _ in range(2)]
    d_loss = torch.ones(1, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    for b, out, s in zip(bs, outs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            b.route(ctx, balance=True, stream=s.cuda_stream)
            b.backward(ctx, out, b.expert, None, d_loss, stream=s.cuda_stream)
        graphs.append(g)
    for _ in range(3):
        for b in bs:
            b.logits.copy_(torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32)))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for b, out in zip(bs, outs):
            ref = Reference(b.seen()[0])
            check_route(b, ref)
            check_stats(b, ref)
            d, tol = ref.backward(None, 1.0)
            assert np.all(np.abs(out.cpu().numpy() - d) <= tol)
    assert ctx.status() == fb.OK


def test_decode_step(gpu):
    """A decode step as a program runs it: router rows times x, routing, the layer on the chosen experts, all on one
    captured stream; the layer's output equals the host call's on the routing read back."""
    import torch
    from tests import quant
    hidden, blocks = 2048, (0, 7)
    rng = np.random.default_rng(24)
    with fb.Context(0, hidden) as ctx:
        g = ctx.g
        pool = np.concatenate([fb.synth_slice(g, 1, k) for k in range(8)])
        ctx.pool_load(pool, fb.synth_shared(g, 1, 99))
        for blk in blocks:
            ctx.fill_layer(blk, 0, 5)
        w = rng.standard_normal((513, hidden)).astype(np.float32) * 0.02
        raw = np.stack([fb.encode_row(fb.Q4_K, r) for r in w])
        wd, a = quant.weights(fb.Q4_K, raw, hidden)
        for tokens in (1, 5):
            x = torch.zeros(tokens, hidden, device="cuda")
            y = torch.zeros(tokens, hidden, device="cuda")
            logits = torch.zeros(tokens, 513, device="cuda")
            expert = torch.zeros(tokens, 10, dtype=torch.int16, device="cuda")
            gate = torch.zeros(tokens, 11, device="cuda")
            m = ctx.matrix(fb.Q4_K, 513, hidden, raw)

            def step(s):
                m.matvec_device(tokens, x.data_ptr(), logits.data_ptr(), stream=s)
                ctx.route_device(tokens, 512, logits.data_ptr(), expert.data_ptr(), gate.data_ptr(),
                                 flags=fb.ROUTE_SHARED, stream=s)
                ctx.run_device(0, tokens, expert.data_ptr(), gate.data_ptr(), x.data_ptr(), None, None,
                               y.data_ptr(), fb.ACT_Q8, 0, s)

            side = torch.cuda.Stream()
            step(side.cuda_stream)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step(side.cuda_stream)
            for _ in range(2):
                xh = rng.standard_normal((tokens, hidden)).astype(np.float32)
                x.copy_(torch.from_numpy(xh))
                graph.replay()
                torch.cuda.synchronize()
                assert ctx.status() == fb.OK
                lo = logits.cpu().numpy().astype(np.float64)
                tol = (hidden / 8 + hidden / 128 + 16) * 2.0 ** -23 * (np.abs(xh).astype(np.float64) @ a.T) \
                    + 2.0 ** -34 * np.abs(xh).max() * a.sum(1)
                assert np.all(np.abs(lo - xh.astype(np.float64) @ wd.T) <= tol)
                ref = Reference(lo[:, :512], None, lo[:, 512])
                assert np.array_equal(expert.cpu().numpy(), ref.expert)
                e, gt = expert.cpu().numpy().astype(np.uint16), gate.cpu().numpy()
                assert np.all(np.abs(gt[:, :10] - ref.g) <= (2 * ref.Rg + 20) * U * ref.g)
                rc, host = ctx.run(0, e, gt, xh, fb.ACT_Q8)
                assert rc == fb.OK
                assert np.array_equal(y.cpu().numpy().view(np.uint32), host.view(np.uint32))
            del graph
            m.close()


def gradient(ctx, b, d_gate, d_loss=None, expert=None):
    """The gradient's columns [T][E (+ 1)] as float64, for d_gate [T][11] (numpy or None)."""
    import torch
    out = torch.full((b.T, b.cols), 5.0, dtype=b.logits.dtype, device="cuda")
    dg = None if d_gate is None else torch.from_numpy(np.ascontiguousarray(d_gate, np.float32)).cuda()
    dl = None if d_loss is None else torch.full((1,), d_loss, device="cuda")
    b.backward(ctx, out, b.expert if expert is None else expert, dg, dl)
    torch.cuda.synchronize()
    return out.float().cpu().numpy().astype(np.float64)


BOTH_TYPES_AND_LOSSES = pytest.mark.parametrize("dtype,d_loss", [(fb.F32, None), (fb.F32, -0.5), (fb.BF16, None), (fb.BF16, -0.5)])
NOT_NUMBERS = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("T,E", [(1, 10), (37, 512), (300, 97)])
@BOTH_TYPES_AND_LOSSES
def test_shared_gradient_stays_in_its_column(ctx, T, E, dtype, d_loss):
    """What d_gate[t][10] holds reaches no expert's column: without the shared column it is not looked at, with it a
    value that is not finite stays there."""
    rng = np.random.default_rng(T + E)
    dg = rng.standard_normal((T, 11))
    for value in NOT_NUMBERS:
        b = Buffers(rng.standard_normal((T, E)), dtype)
        b.route(ctx, balance=True)
        dg[:, 10] = 0
        want = gradient(ctx, b, dg, d_loss)
        dg[:, 10] = value
        assert np.array_equal(gradient(ctx, b, dg, d_loss), want)
        b = Buffers(rng.standard_normal((T, E)), dtype, shared=rng.standard_normal(T))
        b.route(ctx, balance=True)
        dg[:, 10] = rng.standard_normal(T)
        want = gradient(ctx, b, dg, d_loss)
        dg[T // 2, 10] = value
        got = gradient(ctx, b, dg, d_loss)
        assert np.array_equal(got[:, :E], want[:, :E])
        assert np.array_equal(np.delete(got[:, E], T // 2), np.delete(want[:, E], T // 2))
        assert not np.isfinite(got[T // 2, E])
        assert ctx.status() == fb.OK


@pytest.mark.parametrize("T,E", [(3, 10), (37, 512), (300, 97)])
@BOTH_TYPES_AND_LOSSES
def test_gradient_of_padding(ctx, T, E, dtype, d_loss):
    """Padding rows get zeros in every column whatever their d_gate, ids and logits hold."""
    import torch
    rng = np.random.default_rng(T * 3 + E)
    valid = rng.random(T) < 0.6
    valid[1] = False
    for value in NOT_NUMBERS:
        l, sh = rng.standard_normal((T, E)), rng.standard_normal(T)
        l[~valid], sh[~valid] = value, value
        b = Buffers(l, dtype, valid=valid, shared=sh)
        b.route(ctx, balance=True)
        dg = rng.standard_normal((T, 11))
        want = gradient(ctx, b, np.where(valid[:, None], dg, 0), d_loss)
        dg[~valid] = value
        ids = b.expert.clone()
        ids[torch.from_numpy(~valid).cuda()] = -1
        got = gradient(ctx, b, dg, d_loss, ids)
        assert ctx.status() == fb.OK
        assert not got[~valid].any()
        assert np.array_equal(got, want) and np.isfinite(got).all()


@pytest.mark.parametrize("T,E", [(3, 10), (37, 512), (300, 97)])
@BOTH_TYPES_AND_LOSSES
def test_gradient_of_a_shared_logit_that_is_nan(ctx, T, E, dtype, d_loss):
    """A NaN shared logit is reported, as in the selection, and its gate is the constant 0; infinite ones are gates of
    0 and 1; where no gate gradient is asked for, it is not looked at."""
    rng = np.random.default_rng(T * 5 + E)
    l, sh = rng.standard_normal((T, E)), rng.standard_normal(T)
    dg = rng.standard_normal((T, 11))
    clean = Buffers(l, dtype, shared=sh)
    clean.route(ctx, balance=True)
    want = gradient(ctx, clean, dg, d_loss)
    assert ctx.status() == fb.OK
    want[1, E] = 0
    for value, status in [(float("nan"), fb.NUMERIC), (float("inf"), fb.OK), (-float("inf"), fb.OK)]:
        sh[1] = value
        b = Buffers(l, dtype, shared=sh)
        b.route(ctx, balance=True)
        assert ctx.status() == status
        got = gradient(ctx, b, dg, d_loss)
        assert ctx.status() == status
        assert np.array_equal(got, want)
        dg[1, 10] = float("nan")
        got = gradient(ctx, b, dg, d_loss)
        assert ctx.status() == status
        assert np.array_equal(got, want)
        dg[1, 10] = 1
        gradient(ctx, b, None, 1.0)
        assert ctx.status() == fb.OK


@pytest.mark.parametrize("T,E", [(9, 10), (40, 512), (300, 97)])
@BOTH_TYPES_AND_LOSSES
def test_gradient_of_masked_gates(ctx, T, E, dtype, d_loss):
    """The gate of a masked expert (or of an id that is none) is the constant 0: its d_gate is not looked at."""
    import torch
    rng = np.random.default_rng(T * 7 + E)
    for value in NOT_NUMBERS:
        b = Buffers(logits_of("few", T, E, rng), dtype)
        b.route(ctx, balance=True)
        chosen = np.take_along_axis(b.seen()[0], b.expert.cpu().numpy().astype(np.int64), 1)
        masked = np.isneginf(chosen)
        assert masked.any(1).all()
        dg = rng.standard_normal((T, 11))
        dg[:, :10][masked] = 0
        want = gradient(ctx, b, dg, d_loss)
        dg[:, :10][masked] = value
        got = gradient(ctx, b, dg, d_loss)
        assert ctx.status() == fb.OK
        assert np.array_equal(got, want) and np.isfinite(got).all()
    b = Buffers(rng.standard_normal((T, E)), dtype)
    b.route(ctx, balance=True)
    dg = rng.standard_normal((T, 11))
    ids = b.expert.clone()
    ids[T // 2, 3] = E
    dg[T // 2, 3] = 0
    want = gradient(ctx, b, dg, d_loss, ids)
    assert ctx.status() == fb.INVALID
    dg[T // 2, 3] = float("nan")
    got = gradient(ctx, b, dg, d_loss, ids)
    assert ctx.status() == fb.INVALID
    assert np.array_equal(got, want) and np.isfinite(got).all()


@pytest.mark.parametrize("dtype", [fb.F32, fb.BF16])
def test_gradient_of_saturated_shared_gates(ctx, dtype):
    """s (1 - s) to a relative bound at every size of the shared logit l.  As e / (1 + e)^2, e = exp(-|l|): e is off by
    2 steps (4 u), 1 + e by u and at most the 4 u of e, a reciprocal by 2 u, twice, and three products: at most
    4 + 2 (1 + 4 + 2) + 3 = 21 u."""
    sh = np.concatenate([np.linspace(-104, 104, 417), [-17.0, 17.0, 1e-3, -1e-3, 0.0, -3e38, 3e38]])
    T, E = sh.size, 10
    rng = np.random.default_rng(2)
    b = Buffers(rng.standard_normal((T, E)), dtype, shared=sh)
    b.route(ctx)
    dg = rng.standard_normal((T, 11)).astype(np.float32).astype(np.float64)
    got = gradient(ctx, b, dg)[:, E]
    assert ctx.status() == fb.OK
    e = np.exp(-np.abs(b.seen()[1]))
    want = e / (1 + e) ** 2 * dg[:, 10]
    tol = 21 * U * np.abs(want) + TINY * (1 + np.abs(dg[:, 10])) + (2.0 ** -8 * np.abs(want) if dtype == fb.BF16 else 0)
    assert np.all(np.abs(got - want) <= tol), (np.abs(got - want) / tol).max()


# rows of each call, more of them than the gradient's launch has warps (3,552 with the balance term on 148 SMs, 7,104
# without): some warps take one row more than others
MANY = [(5000, 512, False, fb.F32, 0), (16391, 512, True, fb.F32, 0), (16391, 512, False, fb.BF16, 0),
        (5003, 512, True, fb.BF16, 0), (9001, 511, True, fb.F32, 0), (5003, 300, False, fb.F32, 0),
        (7200, 301, True, fb.BF16, 2), (15001, 37, False, fb.F32, 1), (11111, 64, True, fb.BF16, 0),
        (6001, 264, False, fb.BF16, 0)]


@pytest.mark.parametrize("T,E,shared,dtype,pad", MANY)
def test_gradient_of_many_rows(ctx, T, E, shared, dtype, pad):
    """Each gradient alone and both, with d_gate, ids, logits and validity of every row its own, out of place and in
    place, rows 16-byte aligned and not."""
    import torch
    rng = np.random.default_rng(T + E)
    valid = rng.random(T) < 0.8
    l = logits_of("normal", T, E, rng)
    l[rng.random((T, E)) < 0.05] = -np.inf
    b = Buffers(l, dtype, pad=pad, valid=valid, shared=rng.standard_normal(T) * 3 if shared else None)
    ref = Reference(b.seen()[0], valid, b.seen()[1])
    b.route(ctx, balance=True)
    dg = rng.standard_normal((T, 11)).astype(np.float32)
    dg[~valid] = np.nan
    d_gate, d_loss = torch.from_numpy(dg).cuda(), torch.full((1,), 0.5 * T, device="cuda")
    dg[~valid] = 0
    for use_gate, use_loss in [(True, True), (True, False), (False, True)]:
        args = (b.expert if use_gate else None, d_gate if use_gate else None, d_loss if use_loss else None)
        out = torch.full((T, b.stride), 5.0, dtype=b.logits.dtype, device="cuda")
        b.backward(ctx, out, *args)
        assert ctx.status() == fb.OK
        d, tol = ref.backward(dg.astype(np.float64) if use_gate else None, 0.5 * T if use_loss else None, shared)
        got = out.float().cpu().numpy().astype(np.float64)
        tol = tol + (2.0 ** -8 * np.abs(d) + 2.0 ** -133 if dtype == fb.BF16 else 0)
        assert np.all(np.abs(got[:, :b.cols] - d) <= tol), (np.abs(got[:, :b.cols] - d) / tol).max()
        assert not got[~valid, :b.cols].any() and np.all(got[:, b.cols:] == 5)
        keep = b.logits.clone()
        b.backward(ctx, b.logits, *args)
        assert ctx.status() == fb.OK
        assert torch.equal(b.logits[:, :b.cols], out[:, :b.cols])
        b.logits.copy_(keep)


@pytest.mark.parametrize("kind", ["normal", "ties", "few"])
@pytest.mark.parametrize("T,E,shared,dtype,pad", MANY)
def test_selection_of_many_rows(ctx, kind, T, E, shared, dtype, pad):
    """Selection and statistics where each warp takes several rows: rows with a shared column behind 512 experts
    (their neighbours lie 513 elements apart) and other rows that are not 16-byte aligned, beside aligned ones."""
    rng = np.random.default_rng(T * 3 + E)
    valid = rng.random(T) < 0.8
    b = Buffers(logits_of(kind, T, E, rng), dtype, pad=pad, valid=valid, shared=rng.standard_normal(T) * 3 if shared else None)
    l, sh = b.seen()
    ref = Reference(l, valid, sh)
    b.route(ctx)
    assert ctx.status() == fb.OK
    check_route(b, ref)
    ids = b.expert.clone()
    b.expert.fill_(-1)
    b.gate.fill_(float("nan"))
    b.route(ctx, balance=True)
    assert ctx.status() == fb.OK
    check_route(b, ref)
    check_stats(b, ref)
    b.count.fill_(-1)
    b.prob.fill_(-1)
    b.stats(ctx, ids)
    assert ctx.status() == fb.OK
    check_stats(b, ref)


@pytest.mark.parametrize("T,E", [(9, 10), (40, 512)])
def test_gradient_of_large_gate_gradients(ctx, T, E):
    """d_gate near the largest fp32 number: g (d - sum g d) is below twice a half of it, and comes out finite."""
    rng = np.random.default_rng(T + E)
    b = Buffers(rng.standard_normal((T, E)) * 0.1)
    ref = Reference(b.seen()[0])
    b.route(ctx)
    dg = (rng.choice((-1, 1), (T, 11)) * rng.uniform(2e38, 3.4e38, (T, 11))).astype(np.float32)
    dg[0] = 3.4e38
    dg[1] = -3.4e38
    got = gradient(ctx, b, dg)
    assert ctx.status() == fb.OK
    want, tol = ref.backward(dg.astype(np.float64))
    assert np.all(np.abs(got - want) <= tol), (np.abs(got - want) / tol).max()
