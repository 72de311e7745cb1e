"""Operators of requests that share a prompt, against their definitions in 64 bits (GPU).

Linear attention tolerance.  u is half a step of the inputs' type relative to the value
(bf16 2^-8, f16 2^-11, f32 2^-24).  In chunks the weights P and the copy of the state are
rounded once to bf16 (at most u times the sums over magnitudes, ``size``) and the outputs once
more (u |o|); exponents and fp32 sums add less than a tenth of that.  Token by token only the
outputs are rounded to the type, the sums are fp32: 2^-23 for each of the tokens and of the
Dk products.  The state is fp32 everywhere: 128 products of three bf16 parts each, summed in
fp32, are within 384 * 2^-23 (below 6e-5) of the sums over magnitudes.
Adjusted logits: a handful of fp32 operations, each off by at most 2^-24 of the magnitudes
added up so far, then one rounding to the type.
Whole numbers (pages, lengths, lists) have to be equal.
"""

from __future__ import annotations

import random
import threading

import pytest
import torch

from local_kimi_b200 import _lib, ops
from local_kimi_b200.speculative import PagedCache
from oracle import sharing as ref

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
INF, NAN = float("inf"), float("nan")


def sums(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def ints(values, cuda, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=cuda)


# ---------------------------------------------------------------------------
# linear attention
# ---------------------------------------------------------------------------


def room_of(dtype, out, size, tokens, dk, chunks):
    u = U[dtype]
    fp32 = (tokens + dk) * 2.0 ** -23 * size
    return u * out.abs() + (1.1 * u * size if chunks else fp32) + 1e-7 + (
        2.0 ** -25 if dtype == torch.float16 else 0.0)


def assert_within(got, want, room, what):
    bad = ~((got.double().cpu() - want).abs() <= room)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {bad.nonzero()[0].tolist()}:"
        f" {float(got.cpu()[tuple(bad.nonzero()[0])])} for {float(want[tuple(bad.nonzero()[0])])}")


def linear_inputs(lens, h, hq, hk, dk, dv, dtype, seed, per_token=True, slots=None):
    gen = torch.Generator().manual_seed(seed)
    t = sum(lens)
    q = torch.randn(t, hq, dk, generator=gen).to(dtype)
    k = (torch.randn(t, hk, dk, generator=gen) * dk ** -0.5).to(dtype)
    v = torch.randn(t, h, dv, generator=gen).to(dtype)
    g = -torch.rand(*((t, h) if per_token else (h,)), generator=gen).pow(4) * 3
    s = torch.randn(len(lens) if slots is None else slots, h, dk, dv, generator=gen)
    return q, k, v, g, s


def check_linear(cuda, q, k, v, g, s, lens, longest=None, scale=None):
    dk, dtype = q.shape[2], q.dtype
    scale = dk ** -0.5 if scale is None else scale
    want, size, end, weight = ref.linear_attention(q, k, v, g, sums(lens), scale, s)
    state = None if s is None else s.to(cuda)
    longest = max(lens) if longest is None else longest
    out = ops.linear_attention(q.to(cuda), k.to(cuda), v.to(cuda), g.to(cuda),
                               ints(sums(lens), cuda), longest, state=state, scale=scale)
    chunks = dtype == torch.bfloat16 and longest > 8
    assert_within(out, want, room_of(dtype, want, size, max(lens), dk, chunks), "outputs")
    if state is not None:
        step = 6e-5 if chunks else max(lens) * 2.0 ** -23 + 1e-7
        assert_within(state, end, step * weight, "state")
    return out, state


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lens,h,hq,hk,dk,dv", [
    ([1], 1, 1, 1, 64, 64),
    ([5, 1, 0, 17], 4, 4, 4, 128, 128),
    ([130, 3, 127, 128, 129], 4, 2, 1, 128, 64),
    ([257, 31], 6, 3, 6, 64, 128),
    ([300], 3, 1, 3, 96, 80),
    ([64, 200, 1], 2, 1, 2, 40, 72),
    ([9, 40], 5, 5, 5, 8, 8),
    ([385], 2, 2, 2, 128, 128),
])
def test_linear_attention(cuda, dtype, lens, h, hq, hk, dk, dv):
    q, k, v, g, s = linear_inputs(lens, h, hq, hk, dk, dv, dtype, sum(lens) + h)
    check_linear(cuda, q, k, v, g, s, lens)
    check_linear(cuda, q, k, v, g[:1, :].squeeze(0), None, lens, scale=0.3)


def test_linear_attention_in_segments(cuda):
    # Few heads and long requests: their segments' gains are made first.
    for lens, h in (([1500], 1), ([2050, 600, 1, 512], 2), ([1024, 1025], 1)):
        q, k, v, g, s = linear_inputs(lens, h, h, 1, 64, 64, torch.bfloat16, h)
        check_linear(cuda, q, k, v, g * 0.05, s, lens)


def test_linear_attention_segments_in_turns(cuda):
    # More segments than SMs, of requests so uneven that a request's last one is done before its
    # first has begun: that one still starts from the state as it was.
    lens = [6144] + [100] * 7 + [5130] * 3 + [10] * 3
    q, k, v, g, s = linear_inputs(lens, 4, 1, 4, 64, 64, torch.bfloat16, 6)
    check_linear(cuda, q, k, v, g * 0.002, s, lens)


def test_linear_attention_many_units(cuda):
    # More units than SMs: a CTA goes through several.
    lens = [3, 140, 0, 260, 1] * 5
    q, k, v, g, s = linear_inputs(lens, 16, 4, 16, 64, 64, torch.bfloat16, 5)
    check_linear(cuda, q, k, v, g, s, lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,h,hq,hk,dk,dv", [
    (1, 32, 32, 32, 128, 128), (3, 4, 1, 2, 128, 64), (5, 3, 3, 1, 96, 80), (2, 2, 2, 2, 8, 8),
    (40, 16, 4, 16, 64, 128), (7, 1, 1, 1, 40, 24),
])
def test_linear_attention_step(cuda, dtype, b, h, hq, hk, dk, dv):
    q, k, v, g, s = linear_inputs([1] * b, h, hq, hk, dk, dv, dtype, b + h, slots=b + 3)
    order = torch.randperm(b + 3, generator=torch.Generator().manual_seed(b))[:b]
    want, size, end, weight = ref.linear_attention(q, k, v, g, range(b + 1), dk ** -0.5, s[order])
    state = s.to(cuda)
    out = ops.linear_attention_step(state, q.to(cuda), k.to(cuda), v.to(cuda), g.to(cuda),
                                    state_index=order.int().to(cuda))
    assert_within(out, want, room_of(dtype, want, size, 1, dk, False), "outputs")
    assert_within(state[order.to(cuda)], end, 4 * 2.0 ** -24 * weight, "state")
    rest = [i for i in range(b + 3) if i not in order.tolist()]
    assert torch.equal(state.cpu()[rest], s[rest])


@pytest.mark.parametrize("lens", [[40, 3], [6, 2]])
def test_linear_attention_slots(cuda, lens):
    # A negative slot starts from zero and is not kept; one past the pool likewise, recorded.
    q, k, v, g, s = linear_inputs(lens, 2, 2, 2, 64, 64, torch.bfloat16, 1, slots=3)
    _lib.device_errors()
    for slot, bit in ((-1, 0), (3, 4)):
        state = s.to(cuda)
        out = ops.linear_attention(q.to(cuda), k.to(cuda), v.to(cuda), g.to(cuda),
                                   ints(sums(lens), cuda), max(lens), state=state,
                                   state_index=ints([slot, 1], cuda))
        start = torch.stack([torch.zeros_like(s[0]), s[1]])
        want, size, end, weight = ref.linear_attention(q, k, v, g, sums(lens), 0.125, start)
        assert_within(out, want, 3 * room_of(torch.bfloat16, want, size, 40, 64, True), "outputs")
        assert torch.equal(state[0].cpu(), s[0]) and torch.equal(state[2].cpu(), s[2])
        assert_within(state[1], end[1], 6e-5 * weight[1], "state")
        assert _lib.device_errors() == bit


def test_linear_attention_rows_outside_and_empty(cuda):
    q, k, v, g, s = linear_inputs([50], 2, 2, 2, 64, 64, torch.bfloat16, 2, slots=4)
    for longest in (30, 5):
        state = s.to(cuda)
        cu = [3, 3, 3 + min(longest, 20), 33, 33]
        if longest == 5:
            cu = [3, 3, 8, 13, 13]
        out = ops.linear_attention(q.to(cuda), k.to(cuda), v.to(cuda), g.to(cuda),
                                   ints(cu, cuda), longest, state=state)
        assert not out[:cu[0]].any() and not out[cu[-1]:].any()
        assert torch.equal(state[0].cpu(), s[0]) and torch.equal(state[3].cpu(), s[3])
        a, z = cu[0], cu[-1]
        want, size, end, weight = ref.linear_attention(
            q[a:z], k[a:z], v[a:z], g[a:z], [c - a for c in cu], 0.125, s)
        assert_within(out[a:z], want, room_of(torch.bfloat16, want, size, 30, 64, longest > 8)
                      + 1e-5 * size, "outputs")
        assert_within(state, end, 6e-5 * weight, "state")
    empty = ops.linear_attention(q[:0].to(cuda), k[:0].to(cuda), v[:0].to(cuda), g[:0].to(cuda),
                                 ints([0, 0], cuda), 0, state=s.to(cuda))
    assert empty.shape == (0, 2, 64)
    none = ops.linear_attention(q.to(cuda), k.to(cuda), v.to(cuda), g.to(cuda), ints([0], cuda), 9)
    assert none.shape == (50, 2, 64) and not none.any()


@pytest.mark.parametrize("longest", [200, 7])
def test_linear_attention_decays_of_zero_and_above_one(cuda, longest):
    lens = [longest, longest // 2]
    q, k, v, g, s = linear_inputs(lens, 2, 2, 2, 64, 64, torch.bfloat16, 3)
    g[1, 0] = -INF                     # a reset inside a chunk, twice
    g[4, 0] = -200.0
    g[longest, 1] = -INF               # at a request's first token
    g[2, 1] = 0.5                      # no decay: counts as 0
    check_linear(cuda, q, k, v, g, s, lens)
    g[:, 0] = -90.0                    # each next to nothing, their sums far beyond exp's range
    check_linear(cuda, q, k, v, g, s, lens)
    g[:] = 0.0                         # no decay at all
    check_linear(cuda, q, k, v, g, s, lens)


@pytest.mark.parametrize("lens", [[140, 150], [4, 5]])
@pytest.mark.parametrize("which", ["v", "k", "q", "g"])
def test_linear_attention_values_that_are_no_numbers(cuda, lens, which):
    # They reach their own and later tokens of their request, and no others.
    n = sum(lens)
    for at in (lens[0] // 2, lens[0] - 1, 0):
        q, k, v, g, s = linear_inputs(lens, 2, 2, 2, 64, 64, torch.bfloat16, 4)
        clean, clean_state = check_linear(cuda, q, k, v, g, s, lens)
        for bad in (NAN, INF):
            args = dict(q=q.clone(), k=k.clone(), v=v.clone(), g=g.clone())
            args[which][(at, 0, 5) if which != "g" else (at, 0)] = NAN if which == "g" else bad
            state = s.to(cuda)
            out = ops.linear_attention(*(args[x].to(cuda) for x in "qkvg"),
                                       ints(sums(lens), cuda), max(lens), state=state)
            odd = ~torch.isfinite(out)
            hit = torch.zeros(n, 2, 64, dtype=torch.bool, device=cuda)
            cols = slice(5, 6) if which == "v" else slice(None)
            hit[at:(at + 1 if which == "q" else lens[0]), 0, cols] = True
            assert not bool((odd & ~hit).any())
            assert bool(odd[hit].all())
            assert torch.equal(out[~hit], clean[~hit])
            touched = ~torch.isfinite(state)
            keep = torch.zeros_like(touched)
            if which == "v":
                keep[0, 0, :, 5] = True
            elif which == "k":
                keep[0, 0, 5] = True
            elif which == "g":
                keep[0, 0] = True
            assert torch.equal(touched, keep)
            assert torch.equal(state[~keep], clean_state[~keep])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_linear_attention_in_blocks(cuda, dtype):
    # Resets, decays above 1 and far apart, in and across blocks of 32 tokens.
    for lens, h, dk, dv in (([9, 100, 0, 31, 33], 3, 64, 40), ([200], 1, 128, 128)):
        q, k, v, g, s = linear_inputs(lens, h, h, 1, dk, dv, dtype, 17)
        check_linear(cuda, q, k, v, g, s, lens)
        g[::5] = 2.0
        g[7::31, 0] = -INF
        g[33::40] = -150.0
        g[34::9] = -80.0
        g[64] = -INF
        check_linear(cuda, q, k, v, g, s, lens)
    check_linear(cuda, q, k, v, torch.full((200, 1), -103.9), s, lens)
    check_linear(cuda, q, k, v, torch.full((200, 1), -104.1), s, lens)
    check_linear(cuda, q, k, v, torch.zeros(200, 1), s, lens)


@pytest.mark.parametrize("which", ["v", "k", "q", "g"])
def test_linear_attention_no_numbers_in_blocks(cuda, which):
    lens = [70, 50]
    q, k, v, g, s = linear_inputs(lens, 2, 2, 2, 64, 64, torch.float32, 18)
    clean, clean_state = check_linear(cuda, q, k, v, g, s, lens)
    for at in (0, 30, 31, 32, 45, 69):
        for bad in (NAN, INF):
            args = dict(q=q.clone(), k=k.clone(), v=v.clone(), g=g.clone())
            args[which][(at, 0, 5) if which != "g" else (at, 0)] = NAN if which == "g" else bad
            state = s.to(cuda)
            out = ops.linear_attention(*(args[x].to(cuda) for x in "qkvg"),
                                       ints(sums(lens), cuda), max(lens), state=state)
            hit = torch.zeros(120, 2, 64, dtype=torch.bool, device=cuda)
            cols = slice(5, 6) if which == "v" else slice(None)
            hit[at:(at + 1 if which == "q" else 70), 0, cols] = True
            assert torch.equal(~torch.isfinite(out), hit)
            assert torch.equal(out[~hit], clean[~hit])
            keep = torch.zeros_like(state, dtype=torch.bool)
            if which == "v":
                keep[0, 0, :, 5] = True
            elif which == "k":
                keep[0, 0, 5] = True
            elif which == "g":
                keep[0, 0] = True
            assert torch.equal(~torch.isfinite(state), keep)
            assert torch.equal(state[~keep], clean_state[~keep])


def test_linear_attention_blocks_of_many_heads(cuda):
    # Around the lengths from which blocks are used, with more CTAs than SMs and fewer.
    for dtype in (torch.float16, torch.float32):
        for lens, h in (([12, 5], 9), ([13, 5], 9), ([40, 7] * 3, 32), ([41, 7] * 3, 32)):
            q, k, v, g, s = linear_inputs(lens, h, h, h, 16, 64, dtype, 19)
            check_linear(cuda, q, k, v, g, s, lens)


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 64), (128, 128), (40, 72)])
@pytest.mark.parametrize("end", [1, 5, 13, 20, 31, 33, 64, 100, 127, 128])
@pytest.mark.parametrize("whole", [0, 2])
def test_linear_attention_beside_values_that_are_no_numbers(cuda, dk, dv, end, whole):
    # What lies behind a request's end, of the next request or of none, does not reach it, where
    # its last chunk has `end` tokens: with `whole` chunks before, of values that are no numbers in
    # their second and fourth 32 rows, which keep half of the warps that prepare a chunk busy.
    n = 128 * whole + end
    lens = [n, 40, 9]
    q, k, v, g, s = linear_inputs(lens + [150], 3, 3, 3, dk, dv, torch.bfloat16, n, slots=3)
    g *= 0.05
    for c in range(whole):
        v[128 * c + 32:128 * c + 64, 0, 3] = NAN
        v[128 * c + 100:128 * c + 128, 1, 9] = INF
    cu = ints(sums(lens), cuda)
    run = lambda s: (ops.linear_attention(  # noqa: E731
        q.to(cuda), k.to(cuda), v.to(cuda), g.to(cuda), cu, n + 40, state=s), s)
    out, state = run(s.to(cuda))
    for bad in (NAN, INF, -INF):
        for x in (q, k, v):
            x[n:n + 40] = bad
            x[n + 49:] = bad
        g[n:n + 40] = NAN
        g[n + 49:] = NAN
        got, end_state = run(s.to(cuda))
        for a, z in ((got[:n], out[:n]), (got[n + 40:], out[n + 40:]),
                     (end_state[::2], state[::2])):
            assert torch.equal(torch.isfinite(a), torch.isfinite(z))
            assert torch.equal(a[torch.isfinite(a)], z[torch.isfinite(z)])
        assert bool(torch.isnan(got[n:n + 40]).all()) and bool(torch.isnan(end_state[1]).all())
    if not whole:
        assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(state).all())


@pytest.mark.parametrize("dtype,h,dv,longest", [
    (torch.bfloat16, 2, 64, 5), (torch.bfloat16, 160, 80, 8), (torch.bfloat16, 3, 72, 100),
    (torch.bfloat16, 1, 128, 1000), (torch.bfloat16, 80, 64, 129), (torch.float16, 2, 40, 13),
    (torch.float32, 40, 128, 41), (torch.float32, 1, 8, 3),
])
def test_linear_attention_of_longer_requests_than_said(cuda, dtype, h, dv, longest):
    # A request's first max_seqlen tokens count; its other rows are zero.
    lens = [longest, 3 * longest + 70, 0, longest + 1, 2, longest + 300]
    kept = [min(n, longest) for n in lens]
    q, k, v, g, s = (x.to(cuda) for x in linear_inputs(lens, h, h, 1, 64, dv, dtype, longest))
    at = torch.cat([torch.arange(a, a + n) for a, n in zip(sums(lens), kept)]).to(cuda)
    want_state = s.clone()
    want = ops.linear_attention(q[at], k[at], v[at], g[at], ints(sums(kept), cuda), longest,
                                state=want_state)
    junk = [torch.full_like(v, NAN) for _ in range(3)]      # what new memory may hold
    del junk
    out = ops.linear_attention(q, k, v, g, ints(sums(lens), cuda), longest, state=s)
    assert torch.equal(out[at], want) and torch.equal(s, want_state)
    rest = torch.ones(out.shape[0], dtype=torch.bool, device=cuda)
    rest[at] = False
    assert not out[rest].any()


@pytest.mark.parametrize("first", [116, 84, 20])
def test_linear_attention_weights_behind_strong_decays(cuda, first):
    # Each query meets one key, a few tokens before it, and decays that leave next to nothing of
    # what lies before `first`.  Queries, keys and values are powers of two, so a weight's rounding
    # to bf16 (u) is the output's whole error but for the weight's exponent: sums of up to 20
    # logarithms of 150 (base 2) lie below 4096 and are rounded to fp32 by up to 2^-13 each, two
    # of them 2^-12 ln 2 = 0.044 u; the exponential adds 2^-22.
    n, h, b, dk = 128, 32, 12, 128
    gen = torch.Generator().manual_seed(first)
    g = torch.full((b, n, h), -103.9)
    g[:, first:] = -torch.rand(b, n - first, h, generator=gen) * 0.2
    q = torch.zeros(b, n, h, dk)
    k = torch.zeros(b, n, 1, dk)
    k[:, torch.arange(n), 0, torch.arange(n)] = 1.0
    to = [first + (i * 7) % (i - first) if i > first else i for i in range(n)]
    to = [max(j, i - 40) for i, j in enumerate(to)]
    q[:, torch.arange(n), :, torch.tensor(to)] = 1.0
    v = torch.exp2(torch.randint(-2, 3, (b, n, h, 8), generator=gen).float())
    q, k, v = (x.view(b * n, -1, x.shape[-1]).bfloat16() for x in (q, k, v))
    run = g.double().cumsum(1)
    want = torch.exp(run - run[:, to])[..., None] * v.view(b, n, h, 8).double()[:, to]
    out = ops.linear_attention(q.to(cuda), k.to(cuda), v.to(cuda), g.view(b * n, h).to(cuda),
                               ints([n * i for i in range(b + 1)], cuda), n, scale=1.0)
    got, late = out.view(b, n, h, 8).double().cpu(), slice(first, None)
    worst = float(((got - want) / want)[:, late].abs().max())
    assert worst <= 1.05 * 2.0 ** -8, worst * 2.0 ** 8


@pytest.mark.parametrize("n,h,dv", [(128, 2, 64), (2048, 1, 128), (4096, 3, 72), (1024, 160, 64)])
def test_linear_attention_state_to_fp32(cuda, n, h, dv):
    # The state of chunks keeps 24 bits (two bf16 parts of its values would keep 16), in segments
    # and whole.  Each chunk names each key row once, so that few roundings meet in an element; in
    # units of 2^-24 of the magnitudes: an exponential is off by 2 ulp (4), its argument, below 2,
    # by 2^-24 ln 2 (0.7), and a term is a product of two of them (9.4) and its value (2 products,
    # 2), split in three parts (the last is off by 2^-24: 1), summed in fp32 by the tensor cores,
    # which may cut off (3 x 2): 18.4.  What lies before a chunk is multiplied by its decay (4.7,
    # and 1 where segments multiply theirs) and added (1, and 1 more between segments).
    gen = torch.Generator(device=cuda).manual_seed(n)
    c, dk = n // 128, 128
    q = torch.zeros(n, 1, dk, device=cuda).bfloat16()
    k = torch.eye(dk, device=cuda).repeat(c, 1)[:, None].bfloat16()
    v = torch.randn(n, h, dv, generator=gen, device=cuda).bfloat16()
    g = -(0.3 + torch.rand(n, h, generator=gen, device=cuda)) / 160
    state = torch.zeros(1, h, dk, dv, device=cuda)
    ops.linear_attention(q, k, v, g, ints([0, n], cuda), n, state=state)
    run = g.double().view(c, 128, h).cumsum(1)
    terms = (run[:, -1:] - run).exp()[..., None] * v.double().view(c, 128, h, dv)
    high = terms.float().bfloat16().double()
    parts = high + (terms - high).float().bfloat16().double()
    want = torch.zeros(dk, h, dv, dtype=torch.float64, device=cuda)
    size, units, two = want.clone(), want.clone(), want.clone()
    for i in range(c):
        keep = run[i, -1].exp()[:, None]
        units = keep * (units + 5.7 * size)
        two = keep * two + parts[i]
        want, size = keep * want + terms[i], keep * size + terms[i].abs()
        units += 18.4 * terms[i].abs() + 2 * size
    off = (state[0].transpose(0, 1).double() - want).abs()
    assert bool((off <= units * 2.0 ** -24).all()), float((off / size).max())
    # (Two parts alone would not do.)
    assert bool(((two - want).abs() > units * 2.0 ** -24).any())


@pytest.mark.parametrize("dtype,n", [
    (torch.bfloat16, 7), (torch.bfloat16, 300), (torch.bfloat16, 1500), (torch.float16, 100),
    (torch.float32, 100), (torch.float32, 12)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_linear_attention_no_numbers_before_decays_of_zero(cuda, dtype, n, which, bad):
    # 0 times what is no number is none: the same however a prompt is run, wherever in its 32 rows,
    # its chunk or its segment the decay of 0 lies.
    for h, (dk, dv) in ((2, (64, 64)), (160, (128, 40))):
        q, k, v, g, s = linear_inputs([n], h, h, h, dk, dv, dtype, n)
        at = min(n // 3, 70)
        (k if which == "k" else v)[at, 1, 5] = bad
        for reset in (1, 2, 20, 40, 130):
            if at + reset < n:
                g[at + reset] = -INF if reset % 40 else -300.0
        state = s.to(cuda)
        out = ops.linear_attention(q.to(cuda), k.to(cuda), v.to(cuda), g.to(cuda),
                                   ints([0, n], cuda), n, state=state)
        hit, gone = torch.zeros_like(out, dtype=torch.bool), torch.zeros_like(state, dtype=torch.bool)
        if which == "k":
            hit[at:, 1], gone[0, 1, 5] = True, True
        else:
            hit[at:, 1, 5], gone[0, 1, :, 5] = True, True
        assert torch.equal(~torch.isfinite(out), hit)
        assert torch.equal(~torch.isfinite(state), gone)


def test_linear_attention_no_numbers_in_every_chunk(cuda):
    # Chunk after chunk with values that are no numbers, in one piece and in segments.
    lens = [700]
    for h in (2, 160):
        q, k, v, g, s = linear_inputs(lens, h, 1, 1, 64, 128, torch.bfloat16, 14)
        args = [x.to(cuda) for x in (q, k, v, g)]
        state, bad_state = s.to(cuda), s.to(cuda)
        clean = ops.linear_attention(*args, ints([0, 700], cuda), 700, state=state)
        odd = {(3, 0, 5): NAN, (3, 1, 90): INF, (130, 0, 6): -INF, (131, 0, 6): NAN,
               (140, 1, 5): NAN, (255, 0, 127): INF, (256, 1, 0): INF, (390, 0, 64): NAN,
               (511, 0, 65): NAN, (512, 0, 66): NAN, (699, 1, 67): -INF}
        hit = torch.zeros(700, h, 128, dtype=torch.bool, device=cuda)
        for (t, head, col), value in odd.items():
            args[2][t, head, col] = value
            hit[t:, head, col] = True
        out = ops.linear_attention(*args, ints([0, 700], cuda), 700, state=bad_state)
        assert torch.equal(~torch.isfinite(out), hit)
        assert torch.equal(out[~hit], clean[~hit])
        gone = hit[-1][None, :, None, :].expand_as(state)
        assert torch.equal(~torch.isfinite(bad_state), gone)
        assert torch.equal(bad_state[~gone], state[~gone])


@pytest.mark.parametrize("b,h,longest", [
    (1, 4, 8), (1, 4, 9), (592, 4, 5), (592, 4, 6), (593, 4, 5), (593, 4, 6), (593, 4, 8),
    (36, 2, 3), (37, 2, 3), (75, 1, 3),
])
def test_linear_attention_around_its_forms(cuda, b, h, longest):
    # Lengths and heads where another kernel takes over: outputs within the wider tolerance.
    lens = [longest - i % 3 if longest > 2 else longest for i in range(b)]
    q, k, v, g, s = linear_inputs(lens, h, h, 1, 64, 64, torch.bfloat16, b + longest)
    want, size, end, weight = ref.linear_attention(q, k, v, g, sums(lens), 0.125, s)
    state = s.to(cuda)
    out = ops.linear_attention(q.to(cuda), k.to(cuda), v.to(cuda), g.to(cuda),
                               ints(sums(lens), cuda), longest, state=state)
    assert_within(out, want, room_of(torch.bfloat16, want, size, longest, 64, True), "outputs")
    assert_within(state, end, 6e-5 * weight, "state")


def test_linear_attention_views(cuda):
    # Slices of one projection, a transposed batch, decays of another order, expanded tokens.
    gen = torch.Generator(device=cuda).manual_seed(8)
    x = torch.randn(60, 4, 3 * 64 + 8, generator=gen, device=cuda).bfloat16()
    q, k, v = x[..., :64], x[..., 64:128], x[..., 128:192]
    g = -torch.rand(4, 60, generator=gen, device=cuda).T
    s = torch.randn(2, 4, 64, 64, generator=gen, device=cuda)
    cu = ints([0, 25, 60], cuda)
    big = torch.zeros(2, 9, 64, 64, device=cuda)
    part = big[:, 3:7]
    part.copy_(s)
    plain = s.clone()
    a = ops.linear_attention(q, k, v, g, cu, 35, state=part)
    b = ops.linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), g.contiguous(), cu, 35,
                             state=plain)
    assert torch.equal(a, b) and torch.equal(part, plain)
    assert not big[:, :3].any() and not big[:, 7:].any()
    c = ops.linear_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, g, cu, 35,
                             state=s.clone())
    assert torch.equal(c, b)
    one = x[:1, :, :64].expand(6, 4, 64)
    pool = torch.randn(6, 4, 64, 64, generator=gen, device=cuda)
    for call in (lambda t, st: ops.linear_attention_step(st, t, t, t, g[:6]),
                 lambda t, st: ops.linear_attention(t, t, t, g[:6], ints(range(7), cuda), 1, state=st),
                 lambda t, st: ops.linear_attention(t, t, t, g[:6], ints([0, 6], cuda), 20, state=st)):
        s1, s2 = pool.clone(), pool.clone()
        assert torch.equal(call(one, s1), call(one.contiguous(), s2)) and torch.equal(s1, s2)


def test_linear_attention_goes_on_from_its_state(cuda):
    # A prompt in parts, and token by token, ends like the whole.
    q, k, v, g, s = linear_inputs([400], 4, 4, 2, 128, 128, torch.bfloat16, 9)
    want, size, end, weight = ref.linear_attention(q, k, v, g, [0, 400], 128 ** -0.5, s)
    args = [x.to(cuda) for x in (q, k, v, g)]
    state, outs = s.to(cuda), []
    for a, z in ((0, 130), (130, 133), (133, 396)):
        outs.append(ops.linear_attention(*(x[a:z] for x in args), ints([0, z - a], cuda), z - a,
                                         state=state))
    for t in range(396, 400):
        outs.append(ops.linear_attention_step(state, *(x[t:t + 1] for x in args)))
    assert_within(torch.cat(outs), want, room_of(torch.bfloat16, want, size, 400, 128, True),
                  "outputs")
    assert_within(state, end, 1e-4 * weight, "state")


def test_linear_attention_far_offsets(cuda):
    # Values and outputs past 2^31 elements.
    h, dv, lens = 128, 128, [131_200, 150]
    gen = torch.Generator(device=cuda).manual_seed(10)
    t = sum(lens)
    assert lens[0] * h * dv > 2 ** 31
    q = torch.randn(t, 1, 16, generator=gen, device=cuda).bfloat16()
    v = torch.zeros(t, h, dv, dtype=torch.bfloat16, device=cuda)
    v[lens[0]:] = torch.randn(lens[1], h, dv, generator=gen, device=cuda).bfloat16()
    g = -torch.rand(h, generator=gen, device=cuda)
    out = ops.linear_attention(q, q, v, g, ints(sums(lens), cuda), max(lens))
    small = ops.linear_attention(q[lens[0]:], q[lens[0]:], v[lens[0]:], g,
                                 ints([0, lens[1]], cuda), lens[1])
    assert torch.equal(out[lens[0]:], small) and not out[:lens[0]].any()


def test_linear_attention_captured_and_from_threads(cuda):
    q, k, v, g, s = (x.to(cuda) for x in linear_inputs([700, 30], 2, 2, 2, 64, 64, torch.bfloat16, 11))
    cu = ints([0, 700, 730], cuda)
    one = [x[:2] for x in (q, k, v, g)]

    def step(state):
        out = ops.linear_attention(q, k, v, g, cu, 700, state=state)
        return out, ops.linear_attention_step(state, *one)

    a = s.clone()
    first = step(a)
    after = a.clone()
    second = step(a)
    state = s.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(state)
    state.copy_(s)
    graph.replay()
    assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
    assert torch.equal(state, after)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], second[0]) and torch.equal(state, a)
    results: list = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            mine = s.clone()
            for _ in range(5):
                mine.copy_(s)
                out = step(mine)
            torch.cuda.current_stream().synchronize()
            results[i] = (out[0], mine)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(o, first[0]) and torch.equal(m, after) for o, m in results)


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------


def pool_of(rng, requests, page, longest, extra, width_more=1):
    """Lengths, table, free list and head of a random pool without sharing."""
    lens = [rng.choice([0, 1, page, page - 1, 2 * page, rng.randrange(longest + 1)])
            for _ in range(requests)]
    have = [ref.pages_of(n, page) for n in lens]
    total = sum(have) + extra
    ids = list(range(total))
    rng.shuffle(ids)
    at, table = 0, []
    width = max(max(have), 1) + width_more
    for n in have:
        table.append(ids[at:at + n] + [rng.randrange(total)] * (width - n))   # stale past them
        at += n
    head = 3
    return lens, table, ids[:head] + ids[at:], head, total


@pytest.mark.parametrize("seed", range(12))
def test_fork(cuda, seed):
    rng = random.Random(seed)
    page, requests = rng.choice([1, 8, 16, 100]), rng.choice([2, 5, 40, 700])
    lens, table, free, head, _ = pool_of(rng, requests, page, 300, rng.choice([0, 2, 200]))
    pairs = [(rng.randrange(requests), rng.randrange(requests)) for _ in range(rng.randrange(1, 90))]
    if seed % 3 == 0:                   # padding and pairs that cannot be
        pairs += [(-1, 0), (0, -1), (requests, 0), (1, requests + 5)]
        rng.shuffle(pairs)
    src, dst = [p[0] for p in pairs], [p[1] for p in pairs]
    context, held, tab = ints(lens, cuda), ints(lens, cuda), ints(table, cuda)
    want = ref.fork(lens, table, src, dst, free, head, page)
    for _ in range(2):                  # the same call again does the same
        got = ops.paged_fork(context, tab, ints(src, cuda), ints(dst, cuda), ints(free, cuda),
                             ints([head], cuda), page, reserved_lens=held)
        assert context.tolist() == want[0] == held.tolist()
        assert tab.tolist() == want[1]
        assert [x.tolist() for x in got[:3]] == list(want[2:5])
        assert got.free_head.tolist() == [want[5]] and got.missing.tolist() == [want[6]]
    _lib.device_errors()


def test_fork_reports_pairs_that_cannot_be(cuda):
    table, lens = ints([[0, 1], [2, -1], [-1, -1]], cuda), ints([12, 3, 0], cuda)
    _lib.device_errors()
    for src, dst, bit in (([0], [2], 0), ([-1], [2], 0), ([0, 1], [1, 2], 4), ([0, 1], [2, 2], 4),
                          ([0], [3], 4), ([0], [0], 4)):
        ops.paged_fork(lens.clone(), table.clone(), ints(src, cuda), ints(dst, cuda),
                       ints([5, 6], cuda), ints([0], cuda), 8)
        assert _lib.device_errors() == bit
    # Wider than the table: not made, and counted.
    got = ops.paged_fork(ints([17, 0], cuda), ints([[0, 1], [-1, -1]], cuda), ints([0], cuda),
                         ints([1], cuda), ints([5], cuda), ints([0], cuda), 8)
    assert got.missing.item() == 1 and got.free_head.item() == 0


@pytest.mark.parametrize("seed", range(12))
def test_free_and_compact(cuda, seed):
    rng = random.Random(100 + seed)
    page, requests = rng.choice([1, 8, 16, 100]), rng.choice([1, 5, 40, 900])
    lens, table, free, head, total = pool_of(rng, requests, page, 400, rng.choice([0, 7, 900]))
    for _ in range(requests // 3):      # rows that share their first pages
        a, b = rng.randrange(requests), rng.randrange(requests)
        n = min(lens[a], lens[b]) // page
        table[b][:n] = table[a][:n]
    named = {p for row, n in zip(table, lens) for p in row[:ref.pages_of(n, page)]}
    rest = [p for p in range(total) if p not in named]
    rng.shuffle(rest)
    head = total - len(rest)
    free = [0] * head + rest
    if seed % 4 == 3 and lens[0] > page:        # a place that a plan had no page for
        table[0][0] = -1
    keep = [rng.choice([0, n, n, n // 2, n + 5, -3]) for n in lens]
    args = ints(table, cuda), ints(lens, cuda)
    listed = ints(free, cuda)
    want, want_head = ref.free(table, lens, keep, free, head, page)
    for _ in range(2):
        got = ops.paged_free(*args, ints(keep, cuda), listed, ints([head], cuda), page, total)
        assert got.tolist() == [want_head] and listed.tolist() == want
    assert args[0].tolist() == table
    lens = [min(n, max(k, 0)) for n, k in zip(lens, keep)]
    rows, listed_want, head_want, moves = ref.compact(table, lens, want, want_head, page)
    got = ops.paged_compact(args[0], ints(lens, cuda), listed, got, page, total)
    assert got.block_table.tolist() == rows
    assert got.free_pages.tolist() == listed_want and got.free_head.tolist() == [head_want]
    pad = [-1] * (total // 2 - len(moves))
    assert got.copy_from.tolist() == [a for a, _ in moves] + pad
    assert got.copy_to.tolist() == [z for _, z in moves] + pad
    again = ops.paged_compact(got.block_table, ints(lens, cuda), got.free_pages, got.free_head,
                              page, total)
    assert again.copy_from.tolist() == [-1] * (total // 2)
    assert torch.equal(again.block_table, got.block_table)
    assert _lib.device_errors() == 0


def test_free_and_compact_of_a_large_pool(cuda):
    # As many pages as there may be: the first and last ids, one row.
    total = 1 << 19
    table, lens = ints([[total - 1, 0, total - 2, 77]], cuda), ints([4], cuda)
    free = torch.arange(total, dtype=torch.int32, device=cuda)
    head = ints([4], cuda)
    got = ops.paged_free(table, lens, ints([1], cuda), free, head, 1, total)
    assert got.item() == 1 and free[:5].tolist() == [0, 0, 77, total - 2, 4]
    spare = torch.arange(1, total - 1, dtype=torch.int32, device=cuda)
    done = ops.paged_compact(table, lens, spare[spare != 77], ints([0], cuda), 1, total)
    want = ref.compact(table.tolist(), [4], spare[spare != 77].tolist(), 0, 1)
    assert done.block_table.tolist() == want[0] and done.free_pages.tolist() == want[1]


def test_free_without_room_and_pages_past_the_pool(cuda):
    _lib.device_errors()
    free = ints([9, 9, 7], cuda)
    got = ops.paged_free(ints([[5, 1, 3]], cuda), ints([3], cuda), ints([0], cuda), free,
                         ints([2], cuda), 1, 10)
    assert got.item() == 0 and free.tolist() == [3, 5, 7] and _lib.device_errors() == 4
    free = ints([9, 9, 7], cuda)
    got = ops.paged_free(ints([[5, 12, -1]], cuda), ints([3], cuda), ints([0], cuda), free,
                         ints([2], cuda), 1, 10)
    assert got.item() == 1 and free.tolist() == [9, 5, 7] and _lib.device_errors() == 4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (1, 0, 2), (2, 1, 0)])
@pytest.mark.parametrize("page,heads,dk,dv", [(16, 3, 64, 128), (8, 1, 192, 8), (100, 2, 72, 40)])
def test_copy(cuda, dtype, order, page, heads, dk, dv):
    gen = torch.Generator(device=cuda).manual_seed(page)
    pages = 11

    def cache(width):
        sizes = (pages, page, heads)
        x = torch.randn([sizes[i] for i in order] + [width + 8], generator=gen, device=cuda)
        back = [order.index(i) for i in range(3)] + [3]
        return x.to(dtype).permute(back)[..., :width]

    k, v = cache(dk), cache(dv)
    a, z = [0, 9, -1, 4, 5, 2], [1, 10, 3, -1, 6, 7]
    rows = [page, 1, page, page, 0, page - 3]
    for given in (rows, None):
        want = k.clone(), v.clone()
        for i, (s, t) in enumerate(zip(a, z)):
            n = page if given is None else given[i]
            if s >= 0 and t >= 0:
                for x, y in zip((k, v), want):
                    y[t, :n] = x[s, :n]
        ops.paged_copy(k, v, ints(a, cuda), ints(z, cuda),
                       None if given is None else ints(given, cuda))
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    _lib.device_errors()
    ops.paged_copy(k, v, ints([0, pages], cuda), ints([pages, 1], cuda))
    assert torch.equal(k, want[0]) and _lib.device_errors() == 4


def test_copy_of_long_lists_of_padding(cuda):
    k = torch.randn(3000, 1, 2, 8, device=cuda).bfloat16()
    v = k.clone()
    a = torch.full((200_000,), -1, dtype=torch.int32, device=cuda)
    z = a.clone()
    at = torch.randperm(200_000, device=cuda)[:1000]
    a[at] = torch.arange(1000, dtype=torch.int32, device=cuda)
    z[at] = torch.arange(2000, 3000, dtype=torch.int32, device=cuda)
    ops.paged_copy(k, v, a, z)
    assert torch.equal(k[2000:], k[:1000]) and torch.equal(v[2000:], v[:1000])


def test_copy_far_offsets(cuda):
    # Pages past 2^31 elements.
    k = torch.zeros(70_000, 64, 4, 128, dtype=torch.bfloat16, device=cuda)
    v = torch.zeros(70_000, 64, 4, 8, dtype=torch.bfloat16, device=cuda)
    k[1], v[1] = 3.0, 4.0
    ops.paged_copy(k, v, ints([1], cuda), ints([69_999], cuda))
    assert bool((k[69_999] == 3).all()) and bool((v[69_999] == 4).all())
    ops.paged_copy(k, v, ints([69_999], cuda), ints([5], cuda))
    assert bool((k[5] == 3).all()) and float(k.sum(dtype=torch.float64)) == 3 * 3 * 64 * 4 * 128


# ---------------------------------------------------------------------------
# logits
# ---------------------------------------------------------------------------


def check_logits(cuda, seed, dtype, b, v, rows_of, in_place=False, tree=None, parts=None,
                 longest=60, odd=False, offset=0):
    """One call against the definition; ``parts``: which of the arguments are given."""
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    parts = {"history", "prompt", "rep", "pres", "freq", "bias", "mask"} if parts is None else parts
    cu = sums(rows_of)
    rows = cu[-1] + (2 if tree is not None else 0)
    x = (2.5 * torch.randn(rows, v, generator=gen)).to(dtype)
    if odd:
        for value in (NAN, INF, -INF, 0.0):
            x[:, rng.randrange(v)] = value
    lens = [rng.choice([0, 1, longest, rng.randrange(longest + 1)]) for _ in range(b)]
    prompts = [rng.randrange(n + 1) for n in lens]
    words = min(v, 12)
    history = torch.randint(0, words, (b, longest), generator=gen) * ((v - 1) // max(words - 1, 1))
    history[torch.rand(b, longest, generator=gen) < 0.1] = -1
    fl = lambda lo, hi: lo + (hi - lo) * torch.rand(b, generator=gen)  # noqa: E731
    rep, pres, freq = fl(0.7, 1.5), fl(-0.5, 1.0), fl(-0.3, 0.5)
    for p, neutral in ((rep, 1.0), (pres, 0.0), (freq, 0.0)):
        p[::3] = neutral
    n_bias = 9
    ids = torch.randint(-1, min(v, 30), (b, n_bias), generator=gen)
    values = torch.randn(b, n_bias, generator=gen)
    allowed = torch.rand(rows, v, generator=gen) < 0.4
    if rows > 1:
        allowed[1] = False
    packed = torch.zeros(rows, (v + 31) // 32, dtype=torch.int64)
    for t in range(32):
        col = allowed[:, t::32].long()
        packed[:, :col.shape[1]] |= col << t
    packed = torch.where(packed >> 31 != 0, packed - 2 ** 32, packed).int()
    drafted = torch.randint(0, min(v, 20), (rows,), generator=gen)
    masks = [[(1 << (j + 1)) - 1 for j in range(n)] for n in rows_of]
    if tree:
        for row in masks:
            for j in range(1, len(row)):
                row[j] = (1 << j) | row[rng.randrange(max(0, j - 3), j)]
    flat = [m - (1 << 64) if m >> 63 else m for row in masks for m in row] + [-1] * (rows - cu[-1])
    dev = lambda t: t.to(cuda)  # noqa: E731
    kw = {}
    if "history" in parts:
        kw.update(history=dev(history), history_lens=ints(lens, cuda))
    if "prompt" in parts:
        kw.update(prompt_lens=ints(prompts, cuda))
    if "rep" in parts:
        kw.update(repetition=dev(rep))
    if "pres" in parts:
        kw.update(presence=dev(pres))
    if "freq" in parts:
        kw.update(frequency=dev(freq))
    if "bias" in parts:
        kw.update(bias_ids=dev(ids), bias_values=dev(values))
    if "mask" in parts:
        kw.update(allowed=dev(packed))
    if tree is not None:
        kw.update(cu_tokens=ints(cu, cuda), tokens=dev(drafted))
        if tree:
            kw.update(tree_mask=torch.tensor(flat, dtype=torch.int64, device=cuda))
    y = torch.empty(rows * v + offset, dtype=dtype, device=cuda)[offset:].view(rows, v)
    y.copy_(x)
    if in_place:
        kw.update(out=y)
    got = ops.adjust_logits(y, **kw)
    assert (got is y) == in_place
    if not in_place:
        assert torch.equal(y.cpu().view(torch.int16 if dtype != torch.float32 else torch.int32),
                           x.view(torch.int16 if dtype != torch.float32 else torch.int32))
    got = got.double().cpu()
    for i in range(b):
        words_ = history[i, :lens[i]].tolist() if "history" in parts else []
        p = prompts[i] if "prompt" in parts else 0
        for j, r in enumerate(range(cu[i], cu[i + 1])):
            more = []
            if tree is not None:
                more = [int(drafted[cu[i] + a]) for a in range(rows_of[i]) if masks[i][j] >> a & 1]
            want, size = ref.adjust(
                x[r], words_[:p], words_[p:] + more,
                float(rep[i]) if "rep" in parts else 1.0,
                float(pres[i]) if "pres" in parts else 0.0,
                float(freq[i]) if "freq" in parts else 0.0,
                list(zip(ids[i].tolist(), values[i].tolist())) if "bias" in parts else (),
                set(allowed[r].nonzero()[:, 0].tolist()) if "mask" in parts else None)
            here = got[r]
            assert torch.equal(torch.isnan(here), torch.isnan(want)), (i, j)
            fine = torch.isfinite(want)
            assert torch.equal(here[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
            room = U[dtype] * want.abs() + 2.0 ** -20 * size + 1e-37
            bad = fine & ~((here - want).abs() <= room)
            assert not bool(bad.any()), (i, j, bad.nonzero()[0].item(), here[bad][0], want[bad][0])
    for r in range(cu[-1], rows):
        assert torch.equal(got[r][~torch.isnan(got[r])], x[r].double()[~torch.isnan(x[r].double())])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("b,v", [(1, 100), (3, 163_840), (5, 50_257), (2, 33), (4, 1), (3, 1025),
                                 (2, 2_055)])
def test_adjust_logits(cuda, dtype, b, v):
    check_logits(cuda, b + v, dtype, b, v, [1] * b)
    check_logits(cuda, b + v + 1, dtype, b, v, [1] * b, in_place=True, odd=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows_of,v,tree", [
    ([1], 500, False), ([5, 0, 3, 1], 4_001, True), ([64, 7], 1_030, True), ([70, 2], 333, False),
    ([9], 163_840, True),
])
def test_adjust_logits_of_drafted_tokens(cuda, dtype, rows_of, v, tree):
    check_logits(cuda, v, dtype, len(rows_of), v, rows_of, tree=tree)
    check_logits(cuda, v + 1, dtype, len(rows_of), v, rows_of, tree=tree, in_place=True, odd=True,
                 parts={"rep", "freq", "pres"})


@pytest.mark.parametrize("parts", [set(), {"mask"}, {"bias"}, {"history", "rep"},
                                   {"history", "freq"}, {"history", "prompt", "pres"},
                                   {"history", "prompt"}, {"rep"}, {"bias", "mask"}])
def test_adjust_logits_in_parts(cuda, parts):
    for in_place in (False, True):
        check_logits(cuda, 3, torch.bfloat16, 4, 5_003, [1] * 4, parts=parts, in_place=in_place)


def test_adjust_logits_of_unaligned_rows(cuda):
    for offset in (1, 3, 8):
        for in_place in (False, True):
            check_logits(cuda, offset, torch.bfloat16, 3, 2_050, [1] * 3, offset=offset,
                         in_place=in_place)
    x = torch.randn(4, 3000, device=cuda).bfloat16()
    bits = torch.randint(-2 ** 31, 2 ** 31, (4, 63), device=cuda).int()
    wide, narrow = x[:, 5:2005], x[:, 5:2005].contiguous()
    assert torch.equal(ops.adjust_logits(wide, allowed=bits), ops.adjust_logits(narrow, allowed=bits))
    assert torch.equal(ops.adjust_logits(x.T[:4, :4].T.contiguous().T, allowed=bits[:, :1]),
                       ops.adjust_logits(x.T[:4, :4].contiguous(), allowed=bits[:, :1]))
    target = torch.zeros(4, 3000, device=cuda).bfloat16()
    got = ops.adjust_logits(wide, allowed=bits, out=target[:, 500:2500])
    assert torch.equal(got, ops.adjust_logits(narrow, allowed=bits))
    assert not target[:, :500].any() and not target[:, 2500:].any()


def test_adjust_logits_of_expanded_rows(cuda):
    # One grammar, one history and one list of biases for all rows.
    gen = torch.Generator(device=cuda).manual_seed(30)
    for rows, v in ((8, 100), (160, 8_201)):
        x = torch.randn(rows, v, generator=gen, device=cuda).bfloat16()
        words = torch.randint(-2 ** 31, 2 ** 31, (1, (v + 31) // 32), generator=gen,
                              device=cuda).int()
        history = torch.randint(0, v, (1, 50), generator=gen, device=cuda)
        ids = torch.randint(0, v, (1, 6), generator=gen, device=cuda)
        values = torch.randn(1, 6, generator=gen, device=cuda)
        other = dict(history_lens=ints([50 - r % 7 for r in range(rows)], cuda),
                     frequency=torch.full((rows,), 0.5, device=cuda))
        one = dict(history=history, bias_ids=ids, bias_values=values, allowed=words)
        spread = {k: t.expand(rows, -1) for k, t in one.items()}
        copies = {k: t.contiguous() for k, t in spread.items()}
        want = ops.adjust_logits(x, **copies, **other)
        assert torch.equal(ops.adjust_logits(x, **spread, **other), want)
        y = x.clone()
        assert torch.equal(ops.adjust_logits(y, **spread, **other, out=y), want)
        open_ = (words[0, torch.arange(v, device=cuda) // 32]
                 >> (torch.arange(v, device=cuda) % 32)) & 1
        assert torch.equal(torch.isinf(want), (open_ == 0).expand(rows, v))


def test_adjust_logits_long_histories(cuda):
    # Counts far above 16 bits, histories longer than the columns say, ids past the vocabulary.
    _lib.device_errors()
    n = 200_000
    history = torch.zeros(2, n, dtype=torch.long, device=cuda)
    history[1] = torch.arange(n, device=cuda) % 3
    x = torch.zeros(2, 10, device=cuda)
    got = ops.adjust_logits(x, history=history, history_lens=ints([n, 10 * n], cuda),
                            frequency=torch.tensor([1.0, 2.0], device=cuda))
    assert got[0].tolist() == [-float(n)] + [0.0] * 9
    assert got[1, :4].tolist() == [-2.0 * 66_667, -2.0 * 66_667, -2.0 * 66_666, 0.0]
    assert _lib.device_errors() == 0
    history[0, 5] = 10
    ops.adjust_logits(x, history=history, history_lens=ints([9, 9], cuda),
                      frequency=torch.ones(2, device=cuda))
    assert _lib.device_errors() == 8
    many = torch.full((2, 4096), 7, dtype=torch.long, device=cuda)
    got = ops.adjust_logits(x, bias_ids=many, bias_values=torch.ones(2, 4096, device=cuda))
    assert got[:, 7].tolist() == [4096.0] * 2 and float(got.abs().sum()) == 2 * 4096


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_adjust_logits_of_many_rows(cuda, dtype):
    # More wide parts of rows than SMs.
    check_logits(cuda, 21, dtype, 80, 8_211, [1] * 80, longest=90)
    check_logits(cuda, 22, dtype, 80, 8_211, [1] * 80, in_place=True, odd=True, offset=3)
    check_logits(cuda, 23, dtype, 40, 8_211, [4] * 40, tree=True, in_place=True)


@pytest.mark.parametrize("rows", [1, 160])
def test_adjust_logits_history_lengths(cuda, rows):
    # Every token named once or more, by histories that end around the parts they are read in.
    v = 9_001
    gen = torch.Generator(device=cuda).manual_seed(24)
    x = torch.randn(rows, v, generator=gen, device=cuda).bfloat16()
    order = torch.stack([torch.randperm(v, generator=gen, device=cuda) for _ in range(rows)])
    rep = torch.full((rows,), 2.0, device=cuda)
    for n in (1, 255, 256, 1023, 1024, 1025, 2047, 2048, 2049, 3073, 4097, 9_001):
        got = ops.adjust_logits(x, history=order, history_lens=ints([n] * rows, cuda),
                                repetition=rep)
        named = torch.zeros_like(x, dtype=torch.bool).scatter_(1, order[:, :n], True)
        assert torch.equal(got, torch.where(named, torch.where(x > 0, x / 2, x * 2), x)), n


def test_adjust_logits_wide_counts_of_many_rows(cuda):
    rows, v, n = 160, 8_200, 40_000
    history = (torch.arange(n, device=cuda) % 8_193).expand(rows, n).contiguous()
    lens = [n - 7 * r for r in range(rows)]
    got = ops.adjust_logits(torch.zeros(rows, v, device=cuda), history=history,
                            history_lens=ints(lens, cuda), prompt_lens=ints([5] * rows, cuda),
                            frequency=torch.ones(rows, device=cuda))
    for r in (0, 1, 77, 159):
        want = torch.bincount(history[r, 5:lens[r]], minlength=v)
        assert torch.equal(got[r], -want.float())


def test_adjust_logits_far_offsets(cuda):
    rows, v = 14_000, 163_840
    assert rows * v > 2 ** 31
    x = torch.zeros(rows, v, dtype=torch.bfloat16, device=cuda)
    bits = torch.full((rows, v // 32), -1, dtype=torch.int32, device=cuda)
    bits[-1] = 1
    got = ops.adjust_logits(x, allowed=bits, out=x)
    last = got[-1].view(-1, 32)             # one token of each word
    assert not last[:, 0].any() and bool(torch.isinf(last[:, 1:]).all())
    assert not got[:-1].any()


# ---------------------------------------------------------------------------
# together, and on their tensors' streams
# ---------------------------------------------------------------------------


def test_requests_that_share_a_prompt(cuda):
    """One prompt, three continuations, pages given back, the pool compacted: every attention
    as if each request had a cache of its own."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    heads, dk, dv, page, prompt = 2, 64, 64, 16, 75
    width = 40
    cache = PagedCache(4, 40, page, heads, dk, dv, max_pages=width)
    make = lambda n, d: torch.randn(n, heads, d, generator=gen, device=cuda).bfloat16()  # noqa: E731
    told: list = [[make(0, dk), make(0, dv)] for _ in range(4)]

    def write(counts):
        plan = cache.plan(ints(counts, cuda), sum(counts))
        k, v = make(sum(counts), dk), make(sum(counts), dv)
        cache.append(k, v, plan)
        at = 0
        for b, n in enumerate(counts):
            told[b] = [torch.cat((told[b][0], k[at:at + n])), torch.cat((told[b][1], v[at:at + n]))]
            at += n
        q = make(sum(counts), dk)
        out = cache.attend(q, plan, max(counts))
        at = 0
        for b, n in enumerate(counts):
            if n:
                alone = ops.prompt_attention(q[at:at + n], *told[b], ints([0, n], cuda), n,
                                             cu_seqlens_k=ints([0, told[b][0].shape[0]], cuda))
                torch.testing.assert_close(out[at:at + n].float(), alone.float(), atol=2e-2,
                                           rtol=2e-2)
            at += n
        assert plan.missing.item() == 0
        cache.advance(ints(counts, cuda))

    def free_pages():
        return cache.free[cache.head.item():].tolist()

    write([prompt, 0, 0, 30])
    before = len(free_pages())
    got = cache.fork(ints([0, 0, -1], cuda), ints([1, 2, 0], cuda))
    assert got.missing.item() == 0
    assert len(free_pages()) == before - 2          # a last page each, the others shared
    assert cache.table[1, :4].tolist() == cache.table[0, :4].tolist()
    told[1], told[2] = list(told[0]), list(told[0])
    write([3, 20, 1, 0])
    write([1, 1, 18, 2])
    # Request 0 is done: its own pages come back, the shared ones stay.
    cache.release(torch.where(ints([1, 0, 0, 0], cuda) > 0, 0, cache.context))
    told[0] = [make(0, dk), make(0, dv)]
    assert cache.context.tolist() == [0, prompt + 21, prompt + 19, 32]
    shared = cache.table[1, :4].tolist()
    assert not set(shared) & set(free_pages())
    write([5, 4, 0, 7])
    cache.release(ints([5, prompt + 25, 0, 10], cuda))
    told[2] = [make(0, dk), make(0, dv)]
    told[3] = [x[:10] for x in told[3]]
    moves = cache.compact()
    assert int((moves.copy_from >= 0).sum()) > 0
    held = {p for row, n in zip(cache.table.tolist(), cache.reserved.tolist())
            for p in row[:ref.pages_of(n, page)]}
    assert held == set(range(len(held)))
    assert sorted(free_pages()) == list(range(len(held), 40))
    write([2, 3, 9, 1])
    cache.release(ints([0, 0, 0, 0], cuda))
    assert sorted(free_pages()) == list(range(40)) and cache.context.tolist() == [0] * 4
    assert _lib.device_errors() == 0


def test_a_pool_that_runs_out(cuda):
    cache = PagedCache(3, 4, 8, 1, 64, 64)
    cache.plan(ints([20, 0, 0], cuda), 20)
    cache.advance(ints([20, 0, 0], cuda))
    got = cache.fork(ints([0, 0], cuda), ints([1, 2], cuda))
    assert got.missing.item() == 1 and cache.context.tolist() == [20, 20, 0]
    assert cache.head.item() == 4
    cache.release(ints([0, 20, 0], cuda))
    again = cache.fork(ints([1], cuda), ints([2], cuda))
    assert again.missing.item() == 0 and cache.context.tolist() == [0, 20, 20]


def test_a_serving_step_captured(cuda):
    """Fork, release, compaction and adjusted logits in a graph move on with every replay."""
    def make():
        gen = torch.Generator(device=cuda).manual_seed(5)
        cache = PagedCache(4, 30, 8, 1, 64, 64)
        cache.k.copy_(torch.randn(cache.k.shape, generator=gen, device=cuda))
        cache.v.copy_(torch.randn(cache.v.shape, generator=gen, device=cuda))
        return cache

    x = torch.randn(4, 1000, device=cuda).bfloat16()
    history = torch.randint(0, 1000, (4, 64), device=cuda)

    def step(cache):
        cache.plan(ones, 4)
        cache.advance(ones)
        cache.fork(zero, target)
        logits = ops.adjust_logits(x, history=history, history_lens=cache.context,
                                   frequency=penalty)
        cache.release(keep)
        cache.compact()
        return logits

    ones, zero, target = ints([13, 0, 2, 1], cuda), ints([0], cuda), ints([1], cuda)
    keep, penalty = ints([1000, 0, 1000, 2], cuda), torch.ones(4, device=cuda)
    plain, graphed = make(), make()
    step(make())
    graph = torch.cuda.CUDAGraph()
    held = [t.clone() for t in (graphed.table, graphed.context, graphed.reserved, graphed.free,
                                graphed.head)]
    with torch.cuda.graph(graph):
        logits = step(graphed)
    for t, old in zip((graphed.table, graphed.context, graphed.reserved, graphed.free,
                       graphed.head), held):
        t.copy_(old)
    for _ in range(4):
        want = step(plain)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want)
        for a, z in ((plain.table, graphed.table), (plain.context, graphed.context),
                     (plain.free, graphed.free), (plain.head, graphed.head)):
            assert torch.equal(a, z)
        assert torch.equal(plain.k, graphed.k) and torch.equal(plain.v, graphed.v)
