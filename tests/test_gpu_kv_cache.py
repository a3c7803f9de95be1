"""The paged key/value cache on a GPU against plain implementations in 64 bits.

Tolerances are sums of the roundings the kernels make, each at most half a step: u(T) = finfo(T).eps / 2 relative.  The
last one, to the type of the output, is at least half the spacing of subnormal numbers: below the smallest normal
number (fp16: 2^-14) the spacing stays what it is there (2^-24), so a value rounds by up to 2^-25 whatever its size.
  rotary   y = a cos -+ b sin: the cosine and sine are off by 2^-22 at most (angle reduced in 64 bits, remainder in half
           turns rounded to fp32, error 2^-24 pi, and the function's own 2 ulp), two products and a sum round once each:
           (2^-22 + 3 2^-24) (|a| + |b|) <= 2^-21 (|a| + |b|); then u(T) |y|.
  attend   scores: products are exact in fp32, D of them are added up by the tensor core with up to D + 8 roundings or
           truncations of the largest partial sum: d = (D + 8) 2^-23 A with A = scale max_j sum_d |q_d k_jd| (and 2^-21 A
           for the scale's own roundings); with E4M3 rows also the queries' bits below 2^-24 of the row's largest.
           probabilities: relative 2 d + 2^-20 (base-2 exponential, difference of the score and the maximum);
           rounded to the values' type, u(P); sums of n terms in fp32: n / 16 + 64 roundings of 2^-24.
           out: (u(P) + 2 d + 2^-20 + (n / 16 + 64) 2^-24) sum_j p_j |v_j| 2 (numerator and denominator) + u(T) |out|.
  weights  (2 d + 2^-20 + (n / 16 + 64) 2^-24) sum_g p + 2^-23 (|w| + sum_g p).
  lse      d + 2^-20 + 2^-22 |lse|.
"""
import ctypes as C
import math

import pytest

from nv_embedding_cache_b200 import capi

pytestmark = pytest.mark.gpu


def kv():
    from nv_embedding_cache_b200 import kv_cache
    return kv_cache


TYPES = {"bf16": "bfloat16", "f16": "float16", "f32": "float32", "e4m3": "float8_e4m3fn"}


def ty(torch, name):
    return getattr(torch, TYPES[name])


def half_step(torch, name):
    return torch.finfo(ty(torch, name)).eps / 2


SUBNORMAL = {"bf16": 2.0**-134, "f16": 2.0**-25, "f32": 2.0**-150, "e4m3": 2.0**-10}       # half the spacing


def rounding(torch, name, want):
    """How far rounding to a type moves values of these sizes."""
    return (half_step(torch, name) * want.abs()).clamp(min=SUBNORMAL[name])


def gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def within(got, want, tol, what):
    d = (got.double() - want).abs()
    bad = ~(d <= tol)
    bad &= ~((got.double() == want) | (got.isnan() & want.isnan()))      # infinities and NaN have to be alike
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((d / tol.clamp(min=1e-300)).nan_to_num().max()):.3g} of its tolerance"


# ---- rotation ------------------------------------------------------------------------------------
def turned(torch, x, positions, freq, axis, interleaved, sign=1.0):
    """(y, |a| + |b|) in 64 bits for rows x [tokens, heads, width]."""
    x = x.double()
    y, m = x.clone(), torch.zeros_like(x)
    n = freq.numel()
    for i in range(n):
        u, v = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        a = sign * positions[int(axis[i])].double() * float(freq[i])
        c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
        y[:, :, u], y[:, :, v] = x[:, :, u] * c - x[:, :, v] * s, x[:, :, v] * c + x[:, :, u] * s
        m[:, :, u] = m[:, :, v] = x[:, :, u].abs() + x[:, :, v].abs()
    return y, m


def plan_of(torch, pairs, axes, interleaved):
    freq = torch.tensor([10000.0 ** (-i / max(pairs, 1)) for i in range(pairs)], device="cuda")
    axis = torch.tensor([i % axes for i in range(pairs)], dtype=torch.int32, device="cuda")
    return kv().RotaryPlan(freq, axis, axes, interleaved=interleaved), freq, axis


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens,heads,kv_heads,width,pairs,axes,interleaved,far", [
    (1, 1, 1, 2, 1, 1, False, 10), (5, 3, 1, 64, 32, 1, False, 1000), (5, 3, 1, 64, 32, 1, True, 1000),
    (67, 4, 2, 80, 20, 2, False, 100000), (67, 4, 2, 80, 20, 2, True, 100000), (33, 5, 5, 96, 48, 3, False, 2**31 - 1),
    (2, 2, 1, 7, 3, 2, False, 50), (2, 2, 1, 7, 3, 2, True, 50), (300, 8, 2, 128, 64, 3, True, 20000),
    (1300, 16, 2, 128, 64, 4, False, 20000), (9, 2, 2, 256, 64, 1, False, 5), (4, 1, 1, 18, 9, 2, True, 9), (3, 2, 2, 40, 0, 1, False, 9)])
def test_rotary_forward_and_backward(torch_cuda, dtype, tokens, heads, kv_heads, width, pairs, axes, interleaved, far):
    torch = torch_cuda
    g = gen(torch, tokens * 31 + width)
    plan, freq, axis = plan_of(torch, pairs, axes, interleaved)
    pos = torch.randint(0, far, (axes, tokens), generator=g, device="cuda", dtype=torch.int32)
    pos[0, 0] = -3 if far > 100 else 0
    q, k = (torch.randn((tokens, h, width), generator=g, device="cuda").to(ty(torch, dtype)).requires_grad_() for h in (heads, kv_heads))
    gq, gk = (torch.randn(t.shape, generator=g, device="cuda").to(t.dtype) for t in (q, k))
    out = kv().rotary(q, k, pos, plan)
    grads = torch.autograd.grad(out, (q, k), (gq, gk))
    for got, x, sign, name in ((out[0], q, 1, "q"), (out[1], k, 1, "k"), (grads[0], gq, -1, "gq"), (grads[1], gk, -1, "gk")):
        want, m = turned(torch, x.detach(), pos, freq, axis, interleaved, sign)
        assert got.dtype == x.dtype and got.shape == x.shape
        within(got.detach(), want, 2.0**-21 * m + rounding(torch, dtype, want), name)
    plan.check()


def test_rotary_gradient_against_differences(torch_cuda):
    """<g, (f(x + h e) - f(x - h e)) / 2h> for random directions e: the rotation is linear, so the difference is exact
    but for fp32's roundings of f: 2^-21 (|a| + |b|) per value, against h = 1."""
    torch = torch_cuda
    g = gen(torch, 3)
    plan, freq, axis = plan_of(torch, 12, 3, False)
    pos = torch.randint(0, 500, (3, 11), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randn((11, 2, 30), generator=g, device="cuda", requires_grad=True)
    up = torch.randn(x.shape, generator=g, device="cuda")
    grad, = torch.autograd.grad(kv().rotary(x, None, pos, plan), x, up)
    for seed in range(4):
        e = torch.randn(x.shape, generator=gen(torch, 50 + seed), device="cuda")
        with torch.no_grad():
            diff = (kv().rotary(x + e, None, pos, plan).double() - kv().rotary(x - e, None, pos, plan).double()) / 2
        want = float((up.double() * diff).sum())
        tol = float((up.abs().double() * 2.0**-20 * 2 * (x.detach().abs() + e.abs()).double().amax()).sum() + (grad * e).abs().sum() * 2.0**-20)
        assert abs(float((grad.double() * e.double()).sum()) - want) <= tol


def test_rotary_second_derivative_and_no_gradient(torch_cuda):
    """The gradient is linear in the incoming one: its own gradient is the forward rotation."""
    torch = torch_cuda
    g = gen(torch, 4)
    plan, freq, axis = plan_of(torch, 16, 2, True)
    pos = torch.randint(0, 500, (2, 9), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randn((9, 3, 32), generator=g, device="cuda", requires_grad=True)
    up = torch.randn(x.shape, generator=g, device="cuda", requires_grad=True)
    first, = torch.autograd.grad(kv().rotary(x, None, pos, plan), x, up, create_graph=True)
    v = torch.randn(x.shape, generator=g, device="cuda")
    second, = torch.autograd.grad(first, up, v)
    want, m = turned(torch, v, pos, freq, axis, True)
    within(second, want, 2.0**-21 * m + rounding(torch, "f32", want), "second")
    with torch.no_grad():
        out = kv().rotary(x, up, pos, plan)
    assert not out[0].requires_grad and torch.equal(out[0], kv().rotary(x, None, pos, plan).detach())


def test_rotary_strides_broadcasts_and_single_gradients(torch_cuda):
    torch = torch_cuda
    g = gen(torch, 5)
    plan, freq, axis = plan_of(torch, 32, 1, False)
    base = torch.randn((13, 6 * 64 + 3), generator=g, device="cuda")
    for at in (0, 1, 4):                                     # a fused projection's slices, aligned and not
        q = base[:, at:at + 4 * 64].view(13, 4, 64).detach().requires_grad_()
        k = base[:, at:at + 64].view(13, 1, 64).expand(13, 3, 64)
        pos = torch.arange(26, dtype=torch.int32, device="cuda")[::2]
        a, b = kv().rotary(q, k, pos, plan)
        for got, x in ((a, q), (b, k)):
            want, m = turned(torch, x.detach(), pos[None], freq, axis, False)
            within(got.detach(), want, 2.0**-21 * m + 2.0**-24 * want.abs(), "strided")
        grad, = torch.autograd.grad(a.sum(), q)              # an expanded gradient; none for b
        want, m = turned(torch, torch.ones_like(q), pos[None], freq, axis, False, -1.0)
        within(grad, want, 2.0**-21 * m + 2.0**-24 * want.abs(), "gradient")
    shared = torch.randn((13, 1, 64), generator=g, device="cuda", requires_grad=True)
    out = kv().rotary(shared.expand(13, 5, 64), None, pos, plan)
    grad, = torch.autograd.grad(out, shared, torch.ones_like(out))
    want, m = turned(torch, torch.ones((13, 1, 64), device="cuda"), pos[None], freq, axis, False, -1.0)
    within(grad, 5 * want, 5 * (2.0**-21 * m + 2.0**-23 * want.abs()) + 2.0**-22, "shared heads")


def test_rotary_reports_an_axis_that_is_none(torch_cuda):
    torch = torch_cuda
    plan = kv().RotaryPlan(torch.ones(4, device="cuda"), torch.tensor([0, 1, 7, -1], dtype=torch.int32, device="cuda"), 2)
    x = torch.randn((3, 1, 8), device="cuda")
    out = kv().rotary(x, None, torch.ones((2, 3), dtype=torch.int32, device="cuda"), plan)
    assert torch.equal(out[..., [2, 3, 6, 7]], x[..., [2, 3, 6, 7]])      # pairs 2 and 3 did not turn
    with pytest.raises(RuntimeError, match="pair_axis"):
        plan.check()
    plan.check()


def test_rotary_in_place_and_zero_tokens(torch_cuda):
    torch = torch_cuda
    g = gen(torch, 8)
    plan, freq, axis = plan_of(torch, 16, 1, True)
    x = torch.randn((21, 3, 40), generator=g, device="cuda", dtype=torch.float16)
    pos = torch.randint(0, 99, (1, 21), generator=g, device="cuda", dtype=torch.int32)
    want = kv().rotary(x, None, pos, plan)
    args = plan._args(pos, 21, x.device)
    r = capi.HeadRows(x.data_ptr(), x.data_ptr(), 240, 80, 240, 80, 3)
    capi.check(capi.lib.nve_b200_rotary(C.byref(args), capi.DTYPE_FLOAT16, 40, 21, C.byref(r), 1, 0, None))
    torch.cuda.synchronize()
    assert torch.equal(x, want)
    assert kv().rotary(x[:0], x[:0], pos[:, :0], plan)[0].shape == (0, 3, 40)


@pytest.mark.parametrize("tokens,heads,width,pairs", [(40000, 6, 80, 40), (40000, 1, 24, 4), (30011, 7, 40, 20)])
def test_rotary_in_place_turns_every_row_once(torch_cuda, tokens, heads, width, pairs):
    """Many tokens of rows whose items do not divide a block's threads, turned where they are."""
    torch = torch_cuda
    g = gen(torch, 9)
    plan, freq, axis = plan_of(torch, pairs, 1, False)
    x = torch.randn((tokens, heads, width), generator=g, device="cuda", dtype=torch.float16)
    pos = torch.randint(0, 999, (1, tokens), generator=g, device="cuda", dtype=torch.int32)
    want = kv().rotary(x, None, pos, plan)
    args = plan._args(pos, tokens, x.device)
    r = capi.HeadRows(x.data_ptr(), x.data_ptr(), heads * width * 2, width * 2, heads * width * 2, width * 2, heads)
    capi.check(capi.lib.nve_b200_rotary(C.byref(args), capi.DTYPE_FLOAT16, width, tokens, C.byref(r), 1, 0, None))
    torch.cuda.synchronize()
    assert torch.equal(x, want)


# ---- a cache and a batch -------------------------------------------------------------------------
class Batch:
    """A cache whose free memory is NaN (E4M3: its NaN), and sequences with shuffled pages; -1 behind the last page."""

    def __init__(self, torch, lengths, *, heads, width, cache, page, layout="head", spare=0, room=0, seed=0, scales=True):
        self.torch = torch
        g = self.g = gen(torch, seed)
        need = [-(-(n + room) // page) for n in lengths]
        pages = sum(need) + spare + 1
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        shape = (pages, heads, page, width) if layout == "head" else (pages, page, heads, width)
        t = ty(torch, cache)

        def pool():
            x = torch.full(shape, float("nan"), device="cuda").to(t)
            return x.permute(0, 2, 1, 3) if layout == "head" else x

        self.keys, self.values = pool(), pool()
        self.weights = torch.rand((pages, heads, page), generator=g, device="cuda") * 0.1
        self.table = torch.full((len(lengths), max(1, max(need, default=1))), -1, dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.spare = order[at:]
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.k_scale = self.v_scale = None
        if cache == "e4m3" and scales:
            self.k_scale, self.v_scale = (torch.rand(heads, generator=g, device="cuda") * 0.05 + 0.01 for _ in range(2))
        self.page = page
        for b, n in enumerate(lengths):
            if n:
                for pool, big in ((self.keys, 20.0 if cache == "e4m3" else 1.0), (self.values, 20.0 if cache == "e4m3" else 1.0)):
                    self.put(pool, b, torch.arange(n, device="cuda"), (torch.randn((n, heads, width), generator=g, device="cuda") * big).to(t))
        self.cache = kv().PagedKVCache(self.keys, self.values, self.weights, key_scale=self.k_scale, value_scale=self.v_scale)

    def place(self, b, rows, table=None):
        return (self.table if table is None else table)[b].long()[rows // self.page], rows % self.page

    def put(self, pool, b, rows, x):
        p, s = self.place(b, rows)
        bits(self.torch, pool)[p, s] = bits(self.torch, x)

    def rows(self, b, n=None, table=None):
        """(keys, values) [n, heads, width] in 64 bits, scales in."""
        n = int(self.lengths[b]) if n is None else n
        p, s = self.place(b, self.torch.arange(n, device="cuda"), table)
        k, v = (bits(self.torch, t)[p, s].view(t.dtype).double() for t in (self.keys, self.values))
        if self.k_scale is not None:
            k, v = k * self.k_scale.double()[:, None], v * self.v_scale.double()[:, None]
        return k, v

    def row_weights(self, b, n=None, table=None, of=None):
        n = int(self.lengths[b]) if n is None else n
        p, s = self.place(b, self.torch.arange(n, device="cuda"), table)
        return (self.weights if of is None else of)[p, :, s]               # [n, heads]


def bits(torch, t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def raw(torch, t):
    """Comparable whole numbers."""
    t = t.contiguous()
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def check_attend(torch, x, q, dtype, cache, scale, *, accumulate=True, max_length=None, dead=()):
    """Runs the attention and holds everything it gives to 64 bits.  `dead`: (sequence, row) pairs that do not count."""
    before = x.weights.clone()
    out, lse = x.cache.attend(q, x.table, x.lengths, scale=scale, accumulate_weights=accumulate, return_lse=True, max_length=max_length)
    torch.cuda.synchronize()
    n, heads, d = q.shape
    h = x.keys.shape[2]
    group = heads // h
    u_p = half_step(torch, "f16" if cache == "e4m3" else cache)
    touched = before.clone()
    for b in range(n):
        length = int(x.lengths[b])
        live = [r for r in range(length) if (b, r) not in dead]
        if not live:
            assert torch.equal(out[b], torch.zeros_like(out[b])) and bool((lse[b] == -math.inf).all())
            continue
        k, v = x.rows(b)
        idx = torch.tensor(live, device="cuda")
        k, v = k[idx], v[idx]
        p_at, s_at = x.place(b, idx)
        for i in range(h):
            mine = slice(i * group, (i + 1) * group)
            qq = q[b, mine].double()
            score = (qq @ k[:, i].T) * scale
            a = float((qq.abs() @ k[:, i].abs().T).max()) * abs(scale)
            delta = (d + 8) * 2.0**-23 * a + 2.0**-21 * a
            terms = (len(live) / 16 + 64) * 2.0**-24
            want_lse = torch.logsumexp(score, dim=1)
            p = torch.exp(score - want_lse[:, None])
            want = p @ v[:, i]
            size = p @ v[:, i].abs()
            within(out[b, mine], want, (2 * (2 * delta + 2.0**-20 + terms) + u_p) * size + rounding(torch, dtype, want), f"out {b} {i}")
            within(lse[b, mine], want_lse, delta + 2.0**-20 + terms + 2.0**-22 * want_lse.abs(), f"lse {b} {i}")
            if accumulate:
                add = p.sum(dim=0)
                old = before[p_at, i, s_at].double()
                within(x.weights[p_at, i, s_at], old + add, (2 * delta + 2.0**-20 + terms) * 2 * add + 2.0**-23 * (old.abs() + add), f"weights {b} {i}")
                touched[p_at, i, s_at] = x.weights[p_at, i, s_at]
    assert torch.equal(raw(torch, touched), raw(torch, x.weights))          # no other weight changed
    return out, lse


LENGTHS = [0, 1, 63, 64, 65, 200, 513]


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("heads,group,width,page,layout", [
    (2, 1, 64, 16, "head"), (2, 4, 128, 16, "slot"), (1, 8, 128, 1, "head"), (3, 3, 80, 7, "slot"), (1, 16, 96, 100, "head"),
    (2, 17, 64, 64, "head"), (1, 32, 128, 24, "slot"), (1, 64, 32, 16, "head"), (1, 65, 128, 16, "head"), (2, 2, 256, 8, "slot"),
    (1, 20, 192, 16, "head"), (1, 40, 256, 33, "head"), (1, 130, 16, 5, "slot")])
def test_attend(torch_cuda, dtype, cache, heads, group, width, page, layout):
    torch = torch_cuda
    x = Batch(torch, LENGTHS, heads=heads, width=width, cache=cache, page=page, layout=layout, spare=2, seed=width + group)
    q = torch.randn((len(LENGTHS), heads * group, width), generator=x.g, device="cuda").to(ty(torch, dtype))
    check_attend(torch, x, q, dtype, cache, 1.0 / math.sqrt(width))
    x.cache.check()


@pytest.mark.parametrize("width", [8, 24, 40, 72, 136, 248])
def test_attend_widths_of_whole_vectors_only(torch_cuda, width):
    torch = torch_cuda
    x = Batch(torch, [77, 130], heads=2, width=width, cache="bf16", page=9, seed=width)
    q = torch.randn((2, 4, width), generator=x.g, device="cuda").bfloat16()
    check_attend(torch, x, q, "bf16", "bf16", 0.3)


def test_attend_long_and_split(torch_cuda):
    """One long sequence beside short ones: units over many CTAs, CTAs over many units."""
    torch = torch_cuda
    x = Batch(torch, [40001, 3, 0, 900], heads=2, width=128, cache="f16", page=16, seed=4)
    q = torch.randn((4, 8, 128), generator=x.g, device="cuda").half()
    check_attend(torch, x, q, "f16", "f16", 0.088)
    x.cache.check()


def test_attend_many_short_sequences(torch_cuda):
    torch = torch_cuda
    lengths = [(i * 37) % 150 for i in range(300)]
    x = Batch(torch, lengths, heads=4, width=64, cache="bf16", page=16, seed=6)
    q = torch.randn((300, 8, 64), generator=x.g, device="cuda").bfloat16()
    check_attend(torch, x, q, "bf16", "bf16", 0.125)


def test_attend_large_scores_ties_and_one_hot(torch_cuda):
    """Scores of a few hundred (one row takes all), equal scores (all rows alike), and a maximum that grows along the
    length."""
    torch = torch_cuda
    x = Batch(torch, [500, 500], heads=1, width=64, cache="bf16", page=16, seed=7)
    ramp = torch.linspace(-1, 1, 500, device="cuda")[:, None, None].expand(500, 1, 64).bfloat16()
    x.put(x.keys, 0, torch.arange(500, device="cuda"), ramp)
    x.put(x.keys, 1, torch.arange(500, device="cuda"), torch.ones_like(ramp))
    q = torch.ones((2, 2, 64), device="cuda").bfloat16()
    q[:, 1] = -1
    check_attend(torch, x, q, "bf16", "bf16", 4.0)


def test_attend_infinite_and_nan_scores(torch_cuda):
    """-inf scores weigh nothing; a sequence of nothing else is empty; +inf and NaN give NaN, as the formulas do."""
    torch = torch_cuda
    x = Batch(torch, [70, 70, 70, 70], heads=1, width=64, cache="f16", page=16, seed=9)
    q = torch.ones((4, 1, 64), device="cuda").half()
    at = torch.arange(70, device="cuda")
    k = torch.randn((70, 1, 64), generator=x.g, device="cuda").half()
    low = k.clone()
    low[5:9, :, 0] = -math.inf
    x.put(x.keys, 0, at, low)
    x.put(x.keys, 1, at, torch.full_like(k, -math.inf))
    high, nan = k.clone(), k.clone()
    high[3, 0, 0], nan[69, 0, 1] = math.inf, math.nan
    x.put(x.keys, 2, at, high)
    x.put(x.keys, 3, at, nan)
    out, lse = x.cache.attend(q, x.table, x.lengths, scale=0.1, return_lse=True)
    score = low[:, 0].double().sum(dim=1) * 0.1
    assert abs(float(lse[0]) - float(torch.logsumexp(score, 0))) < 1e-4
    assert bool(torch.isfinite(out[0]).all())
    assert bool((out[1] == 0).all()) and float(lse[1]) == -math.inf
    assert bool(out[2].isnan().all()) and bool(out[3].isnan().all()) and bool(lse[3].isnan().all())


def test_attend_scales_of_e4m3_queries(torch_cuda):
    """bf16 queries far outside fp16's range meet E4M3 rows."""
    torch = torch_cuda
    x = Batch(torch, [100, 33], heads=1, width=64, cache="e4m3", page=16, seed=10)
    q = torch.randn((2, 4, 64), generator=x.g, device="cuda").bfloat16()
    q[0, 0] *= 1e20
    q[0, 1] *= 1e-20
    q[1, 2] = 0
    for scale, head in ((1e-21, 0), (1e19, 1), (0.1, 2), (0.1, 3)):
        part = torch.zeros_like(q)
        part[:, head] = q[:, head] if head != 1 else torch.cat((q[:1, 1], torch.zeros_like(q[:1, 1])))
        if head == 0:
            part[1, 0] = 0
        check_attend(torch, x, part, "bf16", "e4m3", scale, accumulate=False)


def test_attend_bad_pages_and_lengths_are_left_out_and_reported(torch_cuda):
    torch = torch_cuda
    x = Batch(torch, [50, 40, 30], heads=2, width=64, cache="bf16", page=8, seed=11)
    x.table[0, 2], x.table[1, 0], x.table[1, 4] = 1 << 30, -7, x.keys.shape[0]
    q = torch.randn((3, 4, 64), generator=x.g, device="cuda").bfloat16()
    dead = {(0, r) for r in range(16, 24)} | {(1, r) for r in [*range(0, 8), *range(32, 40)]}
    # rows of dead pages are never read: give the plain form a page it can index
    clean = x.table.clone()
    launch, x.table = x.table, clean.clamp(0, x.keys.shape[0] - 1)
    attend = x.cache.attend
    x.cache.attend = lambda q, table, lengths, **kw: attend(q, launch, lengths, **kw)
    check_attend(torch, x, q, "bf16", "bf16", 0.125, dead=dead)
    with pytest.raises(RuntimeError, match="page id"):
        x.cache.check()
    x.cache.check()
    lengths = torch.tensor([50, 1000, -4], dtype=torch.int32, device="cuda")
    out = attend(q, clean.clamp(0, x.keys.shape[0] - 1), lengths, max_length=40)
    assert bool((out[2] == 0).all())
    with pytest.raises(RuntimeError, match="length"):
        x.cache.check()


def test_attend_strides_and_max_length(torch_cuda):
    torch = torch_cuda
    x = Batch(torch, [90, 17, 64], heads=2, width=64, cache="bf16", page=16, seed=12)
    fused = torch.randn((3, 1 + 8 * 64 + 9), generator=x.g, device="cuda").bfloat16()
    want = None
    for at in (8, 1):                                        # 16-byte aligned rows of a fused projection, and not
        q = fused[:, 8:8 + 4 * 64].view(3, 4, 64)
        if at == 1:
            moved = torch.empty((3, 1 + 4 * 64), device="cuda", dtype=torch.bfloat16)
            moved[:, 1:] = q.reshape(3, -1)
            q = moved[:, 1:].view(3, 4, 64)
        out, _ = check_attend(torch, x, q, "bf16", "bf16", 0.125, max_length=90)
        assert want is None or torch.equal(out, want)
        want = out
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)  # rows that are not dense
    assert torch.equal(x.cache.attend(turned, x.table, x.lengths, scale=0.125), want)
    wide = torch.full((3, 20), 1 << 29, dtype=torch.int32, device="cuda")
    wide[:, :x.table.shape[1]] = x.table
    assert torch.equal(x.cache.attend(q, wide[:, :x.table.shape[1]], x.lengths, scale=0.125), want)
    x.cache.check()


def test_attend_is_the_same_on_every_run(torch_cuda):
    torch = torch_cuda
    x = Batch(torch, [5000, 77, 1300], heads=2, width=128, cache="bf16", page=16, seed=13)
    q = torch.randn((3, 8, 128), generator=x.g, device="cuda").bfloat16()
    start = x.weights.clone()
    first = None
    for _ in range(5):
        x.weights.copy_(start)
        out, lse = x.cache.attend(q, x.table, x.lengths, accumulate_weights=True, return_lse=True)
        got = [raw(torch, t).clone() for t in (out, lse, x.weights)]
        assert first is None or all(torch.equal(a, b) for a, b in zip(first, got))
        first = got


def test_attend_on_streams_at_once_and_in_graphs(torch_cuda):
    """Calls that overlap do not share scratch: two streams at once, and two captured graphs replayed in turn."""
    torch = torch_cuda
    sides = []
    for seed in (20, 21):
        x = Batch(torch, [3000 + seed, 100], heads=2, width=128, cache="bf16", page=16, seed=seed)
        q = torch.randn((2, 8, 128), generator=x.g, device="cuda").bfloat16()
        sides.append((x, q, x.cache.attend(q, x.table, x.lengths), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (x, q, _, stream) in enumerate(sides):
            with torch.cuda.stream(stream):
                got[i].append(x.cache.attend(q, x.table, x.lengths))
    torch.cuda.synchronize()
    for i, (_, _, want, _) in enumerate(sides):
        assert all(torch.equal(o, want) for o in got[i])
    graphs = []
    for x, q, want, _ in sides:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = x.cache.attend(q, x.table, x.lengths, accumulate_weights=True)
        graphs.append((graph, out, want))
    for _ in range(3):
        for graph, out, _ in graphs:
            out.zero_()
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out, want in graphs)
    x, q, want, _ = sides[0]                                 # a replay follows the lengths, not those of the capture
    x.lengths.copy_(torch.tensor([64, 0], dtype=torch.int32))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], x.cache.attend(q, x.table, x.lengths))


def test_attend_offsets_that_pass_32_bits(torch_cuda):
    """Pages 4 GB and more into the pools."""
    torch = torch_cuda
    pages, page, heads, width = 33000, 64, 8, 128            # 4.3 GB of keys
    keys = torch.zeros((pages, heads, page, width), dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3)
    values = torch.zeros((pages, heads, page, width), dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3)
    x = Batch(torch, [150], heads=heads, width=width, cache="bf16", page=page, seed=14)
    table = torch.tensor([[32999, 5, 32768]], dtype=torch.int32, device="cuda")
    keys[table[0].long()], values[table[0].long()] = x.keys[x.table[0].long()], x.values[x.table[0].long()]
    weights = torch.zeros((pages, heads, page), device="cuda")
    cache = kv().PagedKVCache(keys, values, weights)
    q = torch.randn((1, 16, width), generator=x.g, device="cuda").bfloat16()
    assert torch.equal(cache.attend(q, table, x.lengths, accumulate_weights=True), x.cache.attend(q, x.table, x.lengths))
    assert abs(float(weights.double().sum()) - 16.0) < 1e-3
    new = torch.tensor([[32998, 7]], dtype=torch.int32, device="cuda")
    kept, n = cache.evict(table, x.lengths, new, 100)
    cache.append(x.keys[0, :1], x.values[0, :1], new, n)
    assert torch.equal(keys[7, 36], x.keys[0, 0])
    for h in (0, 7):
        rows = kept[0, h].long()
        assert torch.equal(keys[new[0].long()[torch.arange(100, device="cuda") // 64], torch.arange(100, device="cuda") % 64, h],
                           keys[table[0].long()[rows // 64], rows % 64, h])
    cache.check()


# ---- append --------------------------------------------------------------------------------------
def check_append(torch, x, new, *, q_heads, dtype, cache, pairs, axes, interleaved, offsets=True, pad=0, seed=0):
    g = gen(torch, seed)
    heads, width = x.keys.shape[2:]
    tokens = sum(new) + pad
    k, v, q = (torch.randn((tokens, h, width), generator=g, device="cuda").to(ty(torch, dtype)) for h in (heads, heads, q_heads))
    plan, freq, axis = plan_of(torch, pairs, axes, interleaved)
    pos = torch.randint(0, 9000, (axes, tokens), generator=g, device="cuda", dtype=torch.int32)
    ends = [0]
    for n in new:
        ends.append(ends[-1] + n)
    off = torch.tensor(ends, dtype=torch.int32, device="cuda") if offsets else None
    old = [t.clone() for t in (x.keys, x.values, x.weights)]
    got, lengths = x.cache.append(k, v, x.table, x.lengths, q=q, offsets=off, positions=pos, rotary=plan)
    torch.cuda.synchronize()
    x.cache.check()
    assert lengths.tolist() == [int(a) + b for a, b in zip(x.lengths, new)]
    want_q, m = turned(torch, q, pos, freq, axis, interleaved)
    n = ends[-1]
    within(got[:n], want_q[:n], 2.0**-21 * m[:n] + rounding(torch, dtype, want_q[:n]), "q")
    assert bool((got[n:] == 0).all())
    want_k, mk = turned(torch, k, pos, freq, axis, interleaved)
    for b, count in enumerate(new):
        rows = torch.arange(int(x.lengths[b]), int(x.lengths[b]) + count, device="cuda")
        p, s = x.place(b, rows)
        mine = slice(ends[b], ends[b + 1])
        for pool, want, tol, scale, name in ((x.keys, want_k[mine], 2.0**-21 * mk[mine], x.k_scale, "k"),
                                             (x.values, v[mine].double(), 0.0, x.v_scale, "v")):
            stored = bits(torch, pool)[p, s].view(pool.dtype)
            if scale is not None:
                # the quotient rounds in fp32; a value between two steps may land on either side of the middle
                want, tol = want / scale.double()[:, None], tol / scale.double()[:, None] + 2.0**-23 * (want / scale.double()[:, None]).abs()
                want = want.clamp(-448, 448)
            within(stored.float(), want, tol * (1 + half_step(torch, cache)) + rounding(torch, cache, want), name)
            bits(torch, old[0 if name == "k" else 1])[p, s] = bits(torch, stored)
        assert bool((x.weights[p, :, s] == 0).all())
        old[2][p, :, s] = 0
    for a, b in zip(old, (x.keys, x.values, x.weights)):
        assert torch.equal(raw(torch, a), raw(torch, b))     # nothing else was written
    return lengths


@pytest.mark.parametrize("dtype,cache", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("held,new,heads,q_heads,width,pairs,axes,interleaved,page,layout", [
    ([0], [1], 1, 1, 16, 8, 1, False, 16, "head"), ([5, 0, 33], [1, 1, 1], 2, 8, 128, 64, 1, False, 16, "slot"),
    ([7, 100, 0, 9], [0, 70, 3, 0], 2, 4, 64, 16, 3, True, 7, "head"), ([15, 16, 17], [300, 1, 513], 4, 4, 80, 40, 2, False, 64, "slot"),
    ([3], [2000], 1, 3, 96, 24, 4, True, 33, "head"), ([31, 2], [5, 6], 3, 3, 48, 3, 2, False, 1, "slot"),
    ([31, 2], [5, 6], 3, 3, 48, 7, 2, True, 4, "head"), ([1, 1], [40, 40], 2, 2, 256, 128, 1, False, 16, "slot")])
def test_append(torch_cuda, dtype, cache, held, new, heads, q_heads, width, pairs, axes, interleaved, page, layout):
    torch = torch_cuda
    x = Batch(torch, held, heads=heads, width=width, cache=cache, page=page, layout=layout, room=max(new), seed=width)
    check_append(torch, x, new, q_heads=q_heads, dtype=dtype, cache=cache, pairs=pairs, axes=axes, interleaved=interleaved, pad=3)


def test_append_same_number_each_and_without_rotation(torch_cuda):
    torch = torch_cuda
    x = Batch(torch, [4, 0, 9], heads=2, width=64, cache="bf16", page=4, room=5, seed=30)
    check_append(torch, x, [5, 5, 5], q_heads=4, dtype="bf16", cache="bf16", pairs=32, axes=1, interleaved=False, offsets=False)
    k = torch.randn((3, 2, 64), generator=x.g, device="cuda").bfloat16()
    k[0, 0, 0], k[0, 0, 1] = math.inf, math.nan              # stored as they are
    turned_q, n = x.cache.append(k, -k, x.table, x.lengths)
    assert turned_q is None and n.tolist() == [5, 1, 10]
    for b, row in enumerate((4, 0, 9)):
        p, s = x.place(b, torch.tensor([row], device="cuda"))
        assert torch.equal(raw(torch, x.keys[p, s]), raw(torch, k[b:b + 1])) and torch.equal(raw(torch, x.values[p, s]), raw(torch, -k[b:b + 1]))
    out, n = x.cache.append(k[:0], k[:0], x.table, x.lengths, q=k[:0])
    assert n.tolist() == [4, 0, 9] and out.shape == (0, 2, 64)


def test_append_of_padding_alone(torch_cuda):
    torch = torch_cuda
    x = Batch(torch, [3], heads=1, width=16, cache="bf16", page=4, room=2, seed=33)
    old = [t.clone() for t in (x.keys, x.values, x.weights)]
    k = torch.randn((5, 1, 16), generator=x.g, device="cuda").bfloat16()
    none = torch.zeros((0, 2), dtype=torch.int32, device="cuda")
    q, n = x.cache.append(k, k, none, x.lengths[:0], q=k, offsets=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert n.shape == (0,) and bool((q == 0).all())
    q, n = x.cache.append(k, k, x.table, x.lengths, q=k, offsets=torch.tensor([2, 2], dtype=torch.int32, device="cuda"))
    assert n.tolist() == [3] and bool((q == 0).all())
    for a, b in zip(old, (x.keys, x.values, x.weights)):
        assert torch.equal(raw(torch, a), raw(torch, b))
    # the same through the C ABI without zero_padding: rows of padding are left as they were
    out = torch.full_like(k, 7.0)
    r = capi.HeadRows(k.data_ptr(), out.data_ptr(), 32, 32, 32, 32, 1)
    kv_rows = capi.HeadRows(k.data_ptr(), None, 32, 32, 0, 0, 1)
    off = torch.tensor([1, 3], dtype=torch.int32, device="cuda")
    new = torch.zeros(1, dtype=torch.int32, device="cuda")
    args = capi.KvAppend(capi.DTYPE_BFLOAT16, 5, r, kv_rows, kv_rows, None, x.table.data_ptr(), x.table.stride(0),
                         x.table.shape[1], 1, x.lengths.data_ptr(), off.data_ptr(), new.data_ptr(), 0)
    capi.check(capi.lib.nve_b200_kv_append(C.byref(x.cache._view), C.byref(args), None))
    torch.cuda.synchronize()
    assert new.tolist() == [5] and torch.equal(out[1:3], k[1:3])
    assert bool((out[[0, 3, 4]] == 7.0).all())


def test_refusals_of_the_python_edge(torch_cuda):
    torch = torch_cuda
    x = Batch(torch, [3, 4], heads=2, width=64, cache="bf16", page=4, seed=34, spare=4)
    q = torch.randn((2, 4, 64), device="cuda").bfloat16()
    attend = x.cache.attend
    plan, _, _ = plan_of(torch, 32, 2, False)
    pos = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    k = q[:, :2]
    for call, word in (
            (lambda: attend(q.half(), x.table, x.lengths), "cache's type"), (lambda: attend(q[:1], x.table, x.lengths), "one row"),
            (lambda: attend(q, x.table.long(), x.lengths), "int32"), (lambda: attend(q, x.table, x.lengths.cpu()), "int32"),
            (lambda: attend(q, x.table, x.lengths[:1]), "one row"), (lambda: attend(q[..., :32], x.table, x.lengths), "64"),
            (lambda: attend(q.clone().requires_grad_(), x.table, x.lengths), "gradient"),
            (lambda: x.cache.append(k, k[:1], x.table, x.lengths), "agree"), (lambda: x.cache.append(q, q, x.table, x.lengths), "heads"),
            (lambda: x.cache.append(k, k, x.table, x.lengths, rotary=plan), "together"),
            (lambda: x.cache.append(k, k, x.table, x.lengths, rotary=plan, positions=pos.long()), "int32"),
            (lambda: x.cache.append(k, k, x.table, x.lengths, rotary=plan, positions=pos[:1]), "positions"),
            (lambda: x.cache.append(k, k, x.table, x.lengths, offsets=pos[0]), "one entry more"),
            (lambda: x.cache.append(k, k, x.table, x.lengths, q=q[:1]), "tokens"),
            (lambda: x.cache.evict(x.table, x.lengths, x.table, 0), "budget"), (lambda: x.cache.evict(x.table, x.lengths, x.table, 4, sinks=3, recent=2), "sinks"),
            (lambda: x.cache.evict(x.table, x.lengths, x.table, 1 << 32), "budget"), (lambda: attend(q, x.table, x.lengths, max_length=1000), "max_length"),
            (lambda: attend(q, x.table, x.lengths, max_length=1 << 32), "max_length"), (lambda: attend(q, x.table, x.lengths, max_length=-1), "max_length"), (lambda: x.cache.evict(x.table, x.lengths, x.table[:1], 1), "one row"),
            (lambda: kv().rotary(q, k.half(), pos, plan), "agree"), (lambda: kv().rotary(q.long(), None, pos, plan), "fp32"),
            (lambda: kv().PagedKVCache(x.keys, x.values[:1], x.weights), "match"),
            (lambda: kv().PagedKVCache(x.keys, x.values, x.weights[:1]), "weights"),
            (lambda: kv().PagedKVCache(x.keys, x.values, key_scale=torch.ones(2, device="cuda")), "E4M3")):
        with pytest.raises(ValueError, match=word):
            call()
    for call in (lambda: attend(q[:, :3], x.table, x.lengths),
                 lambda: x.cache.evict(x.table, x.lengths, x.spare[:0].view(2, 0), 5),
                 lambda: kv().PagedKVCache(x.keys, x.values).evict(x.table, x.lengths, x.spare[:2].view(2, 1), 2),
                 lambda: kv().PagedKVCache(x.keys, x.values).attend(q, x.table, x.lengths, accumulate_weights=True)):
        with pytest.raises(capi.NveError):
            call()


def test_append_saturates_and_keeps_nan_in_e4m3(torch_cuda):
    torch = torch_cuda
    x = Batch(torch, [0], heads=1, width=16, cache="e4m3", page=4, room=1, seed=31, scales=False)
    k = torch.zeros((1, 1, 16), device="cuda").half()
    k[0, 0, :4] = torch.tensor([60000.0, -60000.0, math.inf, math.nan], device="cuda")
    x.cache.append(k, k, x.table, x.lengths)
    p, s = x.place(0, torch.tensor([0], device="cuda"))
    got = bits(torch, x.values)[p, s].view(torch.float8_e4m3fn).float().flatten()[:4]
    assert got[:3].tolist() == [448.0, -448.0, 448.0] and bool(got[3].isnan())


def test_append_behind_the_table_and_on_bad_pages(torch_cuda):
    torch = torch_cuda
    x = Batch(torch, [7, 8, 2], heads=1, width=16, cache="bf16", page=4, seed=32)
    table = x.table[:, :2].contiguous()                      # 8 rows each
    table[2, 0] = -1
    old = [t.clone() for t in (x.keys, x.values, x.weights)]
    k = torch.randn((9, 1, 16), generator=x.g, device="cuda").bfloat16()
    q, n = x.cache.append(k, k, table, x.lengths, q=k)
    assert n.tolist() == [8, 8, 5] and torch.equal(q, k)
    with pytest.raises(RuntimeError, match="page id.*length"):
        x.cache.check()
    p, s = int(table[0, 1]), 3                               # the one row that had a place (sequence 2 has no second page)
    old[0][p, s], old[1][p, s], old[2][p, :, s] = k[0], k[0], 0
    if int(table[2, 1]) >= 0:
        p = int(table[2, 1])
        for t, new in ((old[0], k[8]), (old[1], k[8])):
            t[p, 0] = new
        old[2][p, :, 0] = 0
    for a, b in zip(old, (x.keys, x.values, x.weights)):
        assert torch.equal(raw(torch, a), raw(torch, b))


# ---- eviction ------------------------------------------------------------------------------------
def check_evict(torch, x, budget, sinks, recent, new_table, max_length=None):
    old = [t.clone() for t in (x.keys, x.values, x.weights)]
    kept, lengths = x.cache.evict(x.table, x.lengths, new_table, budget, sinks=sinks, recent=recent, max_length=max_length)
    torch.cuda.synchronize()
    assert lengths.tolist() == [min(int(n), budget) for n in x.lengths]
    for b in range(len(x.lengths)):
        length = int(x.lengths[b])
        count = min(length, budget)
        w = x.row_weights(b, of=old[2]).double()
        w = torch.where(w.isnan(), torch.full_like(w, -math.inf), w)
        for h in range(x.keys.shape[2]):
            rank = [(-float(v), i) for i, v in enumerate(w[:, h])]
            fixed = set(range(min(sinks, length))) | set(range(max(0, length - recent), length)) if length > budget else set(range(length))
            others = [i for _, i in sorted(r for r in rank if r[1] not in fixed)]
            want = sorted(fixed | set(others[:count - len(fixed)]))
            assert kept[b, h, :count].tolist() == want, (b, h)
            assert bool((kept[b, h, count:] == -1).all())
            if count:
                src, dst = torch.tensor(want, device="cuda"), torch.arange(count, device="cuda")
                sp, ss = x.place(b, src)
                dp, ds = x.place(b, dst, new_table)
                for t in (old[0], old[1]):
                    bits(torch, t)[dp, ds, h] = bits(torch, t)[sp, ss, h]
                old[2][dp, h, ds] = old[2][sp, h, ss]
    for a, b in zip(old, (x.keys, x.values, x.weights)):
        assert torch.equal(raw(torch, a), raw(torch, b))     # moved as they were, and nothing else written
    return kept, lengths


def new_pages(torch, x, rows):
    per = -(-rows // x.page)
    n = len(x.lengths)
    assert x.spare.numel() >= n * per
    return x.spare[:n * per].view(n, per).contiguous()


@pytest.mark.parametrize("cache", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("lengths,budget,sinks,recent,heads,width,page,layout", [
    ([1], 1, 0, 0, 1, 16, 16, "head"), ([10, 0, 3, 9], 4, 1, 1, 2, 64, 4, "slot"), ([40, 41], 40, 4, 8, 3, 80, 7, "head"),
    ([300, 31, 33, 64], 32, 32, 0, 2, 128, 16, "head"), ([300, 100], 32, 0, 32, 2, 96, 16, "slot"), ([100], 1, 0, 0, 2, 256, 1, "head"),
    ([2500, 1], 700, 3, 50, 2, 32, 24, "slot"), ([5, 6], 1000, 2, 3, 1, 16, 5, "head")])
def test_evict(torch_cuda, cache, lengths, budget, sinks, recent, heads, width, page, layout):
    torch = torch_cuda
    rows = min(budget, max(lengths))
    x = Batch(torch, lengths, heads=heads, width=width, cache=cache, page=page, layout=layout, seed=budget + width,
              spare=len(lengths) * -(-rows // page) + 1)
    x.weights.copy_((x.weights * 40).round() / 40)           # many equal weights
    check_evict(torch, x, budget, sinks, recent, new_pages(torch, x, rows), max_length=max(lengths))
    x.cache.check()


@pytest.mark.parametrize("length,budget", [(9000, 1000), (40000, 39999), (131073, 300)])
def test_evict_long_lists(torch_cuda, length, budget):
    """Lists a cluster shares, with long runs of equal weights over its borders."""
    torch = torch_cuda
    x = Batch(torch, [length], heads=2, width=16, cache="bf16", page=64, seed=length, spare=-(-budget // 64))
    x.weights.copy_(torch.where(x.weights < 0.07, torch.zeros_like(x.weights), x.weights))
    check_evict(torch, x, budget, 4, 100, new_pages(torch, x, budget))


def test_evict_more_rows_than_fit_into_shared_memory(torch_cuda):
    torch = torch_cuda
    x = Batch(torch, [400_001], heads=1, width=16, cache="e4m3", page=128, seed=41, spare=400)
    check_evict(torch, x, 50_000, 1, 7, new_pages(torch, x, 50_000))


def test_evict_weights_out_of_the_ordinary(torch_cuda):
    """Infinities, NaN (as -inf), negative weights, both zeros (alike), subnormals."""
    torch = torch_cuda
    x = Batch(torch, [64], heads=1, width=16, cache="bf16", page=8, seed=42, spare=8)
    odd = [math.inf, -math.inf, math.nan, -0.0, 0.0, -1.0, 1e-42, -1e-42, 3.4e38, -3.4e38, 1.0, 1.0000001]
    p, s = x.place(0, torch.arange(64, device="cuda"))
    x.weights[p, 0, s] = torch.tensor([odd[(i * 5) % len(odd)] for i in range(64)], device="cuda")
    for budget in (1, 5, 20, 30, 40, 50, 60, 63):
        check_evict(torch, x, budget, 0, 0, new_pages(torch, x, budget))


def test_evict_reports_bad_pages_and_leaves_their_rows_out(torch_cuda):
    torch = torch_cuda
    x = Batch(torch, [40], heads=1, width=16, cache="bf16", page=8, seed=43, spare=6)
    table = x.table.clone()
    table[0, 1] = 1 << 20
    new = new_pages(torch, x, 16)
    new[0, 1] = -5
    old = [t.clone() for t in (x.keys, x.values, x.weights)]
    kept, n = x.cache.evict(table, x.lengths, new, 16)
    rows = kept[0, 0].tolist()
    assert n.tolist() == [16] and rows == sorted(set(rows)) and not any(8 <= r < 16 for r in rows)
    with pytest.raises(RuntimeError, match="page id"):
        x.cache.check()
    page = int(new[0, 0])
    for a, b in zip(old, (x.keys, x.values, x.weights)):
        same = raw(torch, a) == raw(torch, b)
        same[page] = True
        assert bool(same.all())


# ---- order on the stream -------------------------------------------------------------------------
def test_calls_follow_what_is_before_them_on_the_stream(torch_cuda):
    """Launches may overlap the end of what runs before them; what they read has to be complete all the same: lengths made
    by a host copy, a fill, another stream or the call before, eager and captured."""
    torch = torch_cuda
    x = Batch(torch, [4000, 4000], heads=4, width=128, cache="bf16", page=16, seed=60, room=200)
    q = torch.randn((2, 8, 128), generator=x.g, device="cuda").bfloat16()
    ends = [torch.tensor(e, dtype=torch.int32, device="cuda") for e in ([4000, 77], [5, 3999])]
    want = [x.cache.attend(q, x.table, e) for e in ends]
    pinned = ends[0].cpu().pin_memory()
    n = torch.zeros(2, dtype=torch.int32, device="cuda")

    def steps(first):
        first()
        a = x.cache.attend(q, x.table, n)
        n.zero_()
        z = x.cache.attend(q, x.table, n)
        n.copy_(ends[1])
        return a, z, x.cache.attend(q, x.table, n)

    def right(a, z, b):
        return torch.equal(a, want[0]) and bool((z == 0).all()) and torch.equal(b, want[1])

    torch.cuda.synchronize()
    got = [steps(lambda: n.copy_(pinned, non_blocking=True)) for _ in range(50)]
    torch.cuda.synchronize()
    assert all(right(*g) for g in got)
    side = torch.cuda.Stream()

    def other_stream():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            n.copy_(ends[0])
        main.wait_stream(side)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = steps(other_stream)
    for _ in range(20):
        for o in out:
            o.fill_(3)
        graph.replay()
    torch.cuda.synchronize()
    assert right(*out)
    k = torch.randn((2, 4, 128), generator=x.g, device="cuda").bfloat16()
    runs = []
    for _ in range(5):
        m, outs = x.lengths, []
        for s in range(30):
            _, m = x.cache.append(k * ((s + 1) / 30), k, x.table, m)
            outs.append(x.cache.attend(q, x.table, m))
        runs.append(torch.stack(outs))
    torch.cuda.synchronize()
    assert m.tolist() == [4030, 4030] and all(torch.equal(runs[0], r) for r in runs)
    x.cache.check()


def test_threads_share_a_cache(torch_cuda):
    """Two host threads, a stream each, the same cache: reads do not disturb one another."""
    import threading
    torch = torch_cuda
    x = Batch(torch, [3000, 500], heads=2, width=128, cache="f16", page=16, seed=61)
    qs = [torch.randn((2, h, 128), generator=x.g, device="cuda").half() for h in (4, 16)]
    want = [x.cache.attend(q, x.table, x.lengths) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            outs = [x.cache.attend(qs[i], x.table, x.lengths) for _ in range(100)]
        stream.synchronize()
        if not all(torch.equal(o, want[i]) for o in outs):
            wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_rotary_backward_in_a_graph(torch_cuda):
    """Forward and gradient captured and replayed on new values.  (No eager graph of the same leaf may be alive then: torch
    keeps the leaf's node on the stream of that one, and refuses the capture for any function.)"""
    torch = torch_cuda
    g = gen(torch, 62)
    plan, freq, axis = plan_of(torch, 32, 2, False)
    pos = torch.randint(0, 500, (2, 50), generator=g, device="cuda", dtype=torch.int32)
    x = torch.randn((50, 4, 64), generator=g, device="cuda", requires_grad=True)
    up = torch.randn(x.shape, generator=g, device="cuda")

    def eager():
        out = kv().rotary(x, None, pos, plan)
        return out.detach(), torch.autograd.grad(out, x, up)[0]

    first = eager()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv().rotary(x, None, pos, plan)
        grad, = torch.autograd.grad(out, x, up)
        out = out.detach()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first[0]) and torch.equal(grad, first[1])
    with torch.no_grad():
        x.mul_(-0.5)
    up.copy_(torch.randn(x.shape, generator=g, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    again = eager()
    assert torch.equal(out, again[0]) and torch.equal(grad, again[1])


# ---- together ------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_a_decode_run_with_eviction(torch_cuda, cache):
    """Prompts go in, tokens are decoded one by one with their attention added up, the cache is pressed to a budget in
    between, and decoding goes on over the new pages: every step against 64 bits on what the cache holds.  The decode
    step is captured once per page table and replayed."""
    torch = torch_cuda
    heads, group, width, page, budget = 2, 4, 64, 16, 48
    plan = kv().RotaryPlan.sections([8, 12, 12])
    x = Batch(torch, [0, 0, 0], heads=heads, width=width, cache=cache, page=page, room=140, spare=3 * 6, seed=50)
    g = gen(torch, 51)
    new = [100, 64, 7]
    ends = torch.tensor([0, 100, 164, 171], dtype=torch.int32, device="cuda")

    def rows(n, h):
        return torch.randn((n, h, width), generator=g, device="cuda").bfloat16()

    pos = torch.randint(0, 100, (3, 171), generator=g, device="cuda", dtype=torch.int32)
    _, lengths = x.cache.append(rows(171, heads), rows(171, heads), x.table, x.lengths, offsets=ends, positions=pos, rotary=plan)
    assert lengths.tolist() == new
    x.lengths = lengths
    table = x.table
    for press in range(2):
        k, v, q = rows(3, heads), rows(3, heads), rows(3, heads * group)
        at = torch.full((3, 3), 100, dtype=torch.int32, device="cuda")
        held = x.lengths.clone()
        state = [t.clone() for t in (x.keys, x.values, x.weights, held)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                        # a first run outside the capture
            x.cache.append(k, v, table, held, q=q, positions=at, rotary=plan)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            turned_q, after = x.cache.append(k, v, table, held, q=q, positions=at, rotary=plan)
            out = x.cache.attend(turned_q, table, after, accumulate_weights=True)
            held.copy_(after)
        for t, s in zip((x.keys, x.values, x.weights, held), state):
            t.copy_(s)
        for step in range(6):
            for t in (k, v, q):
                t.copy_(torch.randn(t.shape, generator=g, device="cuda").bfloat16())
            at.fill_(100 + step)
            before = x.weights.clone()
            graph.replay()
            torch.cuda.synchronize()
            x.lengths, x.table = held.clone(), table
            got, weights = out.clone(), x.weights.clone()
            for b in range(3):                               # the new rows start at weight 0
                p, s = x.place(b, x.lengths[b:b + 1].long() - 1)
                before[p, :, s] = 0
            x.weights.copy_(before)
            again, _ = check_attend(torch, x, turned_q, "bf16", cache, 1.0 / math.sqrt(width))
            assert torch.equal(raw(torch, again), raw(torch, got)) and torch.equal(raw(torch, weights), raw(torch, x.weights))
        if press == 0:
            fresh = x.spare[:18].view(3, 6).contiguous()     # room for the budget and what follows
            kept, lengths = check_evict(torch, x, budget, 4, 16, fresh)
            x.lengths, table = lengths, fresh
            x.table = fresh
    x.cache.check()
