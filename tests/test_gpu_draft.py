"""The operators of speculative decoding against their definitions in 64 bits, on a GPU.

Tolerances are bounds: a rounding to a type is off by at most eps / 2 of the value, an f32 operation by 2^-24 of its result, an
mma that adds to an accumulator by 2^-23 of the largest partial sum.
"""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from dyninfer_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"q8": torch.int8, "e4m3": torch.float8_e4m3fn}


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def normal(seed, *shape):
    return torch.randn(*shape, generator=gen(seed), device="cuda")


def half(t):
    return torch.finfo(t).eps / 2


# ---- rotary -----------------------------------------------------------------------------------------------------------
def rotated(x, angle, rot, layout, magnitude):
    """(result, bound on |difference|): angle [..., rot / 2] in 64 bits, modulo a turn."""
    y = x.double().clone()
    first = slice(0, rot // 2) if layout == "half" else slice(0, rot, 2)
    second = slice(rot // 2, rot) if layout == "half" else slice(1, rot, 2)
    a, b = x.double()[..., first], x.double()[..., second]
    c, s = magnitude * angle.cos()[..., None, :], magnitude * angle.sin()[..., None, :]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    # the angle in f32, up to pi 2^-24; sincospif 2^-23 (its documented one ulp); the magnitude and three operations 2^-24 each
    bound = torch.zeros_like(y)
    bound[..., first] = bound[..., second] = abs(magnitude) * (math.pi + 2 + 4) * 2.0 ** -24 * (a.abs() + b.abs())
    return y, bound + half(x.dtype) * (y.abs() + bound) + (2.0 ** -25 if x.dtype == torch.float16 else 0)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,heads,d,rot", [(1, 1, 2, 2), (5, 24, 128, 128), (7, 3, 80, 34), (33, 5, 256, 256), (300, 40, 128, 64),
                                              (2, 1, 96, 96), (65, 2, 64, 6), (1, 700, 16, 8), (3, 2, 256, 34), (5, 3, 256, 2),
                                              (2, 3, 255, 254)])
def test_rotary(native_lib, layout, kind, rows, heads, d, rot):
    x = normal(rows + d, rows, heads, d).to(TYPES[kind])
    positions = torch.randint(0, 300000, (rows,), generator=gen(3), device="cuda")
    f, m = ops.rotary_frequencies(rot, 1e4)
    m = 1.25 if rot == 64 else m
    want, bound = rotated(x, positions.double()[:, None] * f.cuda(), rot, layout, m)
    got = ops.rotary(x, positions, f, layout, m)
    assert got.dtype == x.dtype and bool(((got.double() - want).abs() <= bound).all())
    assert torch.equal(got[..., rot:], x[..., rot:])


def test_rotary_positions_far_out_and_below_zero(native_lib):
    positions = [0, 1, -1, -12345, 2 ** 24 + 1, 2 ** 40 + 12345, -2 ** 45 + 3]
    f = torch.tensor([1.0, 0.37, 1e-3, 1e-6], dtype=torch.float64)
    # 45 digits of pi: exact enough modulo a turn
    pi = Fraction(3141592653589793238462643383279502884197169399, 10 ** 45)
    angle = [[float((Fraction(p) * Fraction(float(w)) / (2 * pi)) % 1 * 2 * pi) for w in f] for p in positions]
    x = normal(1, len(positions), 3, 8)
    want, bound = rotated(x, torch.tensor(angle, dtype=torch.float64, device="cuda"), 8, "half", 1.0)
    # a fraction of a turn is off by 2^-53 / 2 pi relative (the division in at least 64 bits) and 2^-65: at 2^45 below 1e-5 rad
    bound = bound + torch.tensor([abs(p) * 2.0 ** -63 for p in positions], device="cuda")[:, None, None] * 2 * math.pi * 8
    got = ops.rotary(x, torch.tensor(positions, device="cuda"), f)
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_in_place_on_fused_rows_batched_and_unaligned(native_lib, layout):
    f, _ = ops.rotary_frequencies(128)
    rows = normal(5, 2, 7, 10 * 128).to(torch.bfloat16)
    whole = rows.clone()
    view = whole.view(2, 7, 10, 128)[:, :, :6]          # q and k of [q | k | v]
    positions = torch.arange(14, device="cuda").view(2, 7) * 3
    want = ops.rotary(rows.view(2, 7, 10, 128)[:, :, :6].contiguous(), positions, f, layout)
    assert ops.rotary(view, positions, f, layout, out=view) is view
    assert torch.equal(view, want) and torch.equal(whole[..., 6 * 128:], rows[..., 6 * 128:])
    # part of the head, in place, and a start that is not a multiple of 16 bytes: the same numbers
    f, _ = ops.rotary_frequencies(32)
    x = normal(6, 7 * 3 * 128 + 3)
    odd = x[3:].view(7, 3, 128)
    want = ops.rotary(odd.clone(), positions[0], f, layout)
    assert torch.equal(ops.rotary(odd, positions[0], f, layout), want)
    assert torch.equal(ops.rotary(odd, positions[0].to(torch.int32), f, layout, out=odd), want)
    assert ops.rotary(x[:0].view(0, 3, 128), positions[0][:0], f).shape == (0, 3, 128)


def test_rotary_agrees_with_rope(native_lib):
    """The half layout at consecutive positions is what `ops.rope` does, which rounds its angles to f32: 100 2^-24 at 100."""
    x = normal(7, 100, 4, 128)
    f = (1e6 ** -(torch.arange(64, dtype=torch.float64) * 2 / 128))
    got = ops.rotary(x, torch.arange(100, device="cuda"), f)
    assert float((got - ops.rope(x, 0, 1e6)).abs().max()) <= 2 * float(x.abs().max()) * 3 * 100 * 2.0 ** -24


# ---- the 8-bit cache --------------------------------------------------------------------------------------------------
def quantised(x, kind):
    """(codes as numbers, scale) of rows along the last dimension, from the definition, in 64 bits."""
    x = x.double().cpu().numpy()
    top = np.abs(x).max(-1)
    finite = np.isfinite(top)
    codes, scale = np.zeros(x.shape), np.zeros(top.shape)
    scale[~finite] = np.nan
    used = finite & (top >= 2.0 ** -100)
    for i in np.argwhere(used):
        i = tuple(i)
        if kind == "q8":
            scale[i] = np.float32(top[i] / 127)
            codes[i] = np.round(x[i] * np.float64(np.float32(127 / top[i])))
        else:
            e = math.ceil(math.log2(top[i] / 448))
            while top[i] > 448 * 2.0 ** e:
                e += 1
            while top[i] <= 448 * 2.0 ** (e - 1):
                e -= 1
            scale[i] = 2.0 ** e
            y = x[i] / scale[i]
            unit = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
            codes[i] = np.round(y / unit) * unit
    return codes, scale


def empty_cache(kind, slots, heads, cap, d):
    """A cache full of something else, so that rows written by mistake show."""
    codes = [torch.full((slots, heads, cap, d), 7, dtype=torch.int8, device="cuda").view(CODES[kind]) for _ in "kv"]
    return (*codes, torch.full((slots, heads, cap), 3.0, device="cuda"), torch.full((slots, heads, cap), 3.0, device="cuda"))


def numbers(codes):
    return codes.float().double().cpu().numpy()


@pytest.mark.parametrize("kind", ["q8", "e4m3"])
@pytest.mark.parametrize("source", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("slots,rows,heads,d,cap", [(1, 1, 1, 16, 1), (3, 5, 2, 128, 9), (2, 17, 3, 80, 40), (1, 33, 8, 256, 64),
                                                    (64, 1, 8, 64, 5), (2, 3, 1, 48, 7)])
def test_cache_rows_are_exact(native_lib, kind, source, slots, rows, heads, d, cap):
    k, v = (normal(i, slots, rows, heads, d).to(TYPES[source]) * (1 + i) for i in (11, 12))
    k[..., 0] *= 30                                            # a channel of its own
    starts = torch.arange(slots, device="cuda") % max(1, cap - rows + 1)
    whole = empty_cache(kind, slots, heads, cap, d)
    before = [numbers(whole[0]), numbers(whole[1])]
    ops.kv_write(k, v, starts, *whole)
    for x, codes, scale, old in ((k, whole[0], whole[2], before[0]), (v, whole[1], whole[3], before[1])):
        want_codes, want_scale = quantised(x.permute(0, 2, 1, 3), kind)
        written = np.zeros((slots, heads, cap), bool)
        for b in range(slots):
            at = slice(int(starts[b]), int(starts[b]) + rows)
            written[b, :, at] = True
            assert np.array_equal(numbers(codes)[b, :, at], want_codes[b])
            assert np.array_equal(scale[b, :, at].double().cpu().numpy(), want_scale[b])
        assert np.array_equal(numbers(codes)[~written], old[~written]) and bool((scale.cpu().numpy()[~written] == 3).all())
    for dtype in TYPES.values():
        for x, got in zip((k, v), ops.kv_read(starts, rows, *whole, dtype=dtype)):
            codes, scale = quantised(x, kind)
            want = torch.from_numpy(codes * scale[..., None]).float()         # one rounding to f32, one to the type
            assert got.shape == x.shape and torch.equal(got.cpu(), want.to(dtype))


@pytest.mark.parametrize("kind", ["q8", "e4m3"])
def test_cache_rows_with_extreme_values(native_lib, kind):
    x = normal(3, 1, 12, 1, 32)
    x[0, 0] = 0.0
    x[0, 1, 0, 3] = math.inf
    x[0, 2, 0, 31] = math.nan
    x[0, 3] *= 1e-38
    x[0, 4] = 0.0
    x[0, 4, 0, 5] = 1e-45
    x[0, 5] *= 2.0 ** -99 / x[0, 5].abs().max()
    x[0, 6, 0, 0] = 3.4e38
    x[0, 7] = -2.5                                             # codes -127
    x[0, 8, 0, :] = torch.arange(32, device="cuda") - 15.5     # halves, towards even after a factor of 127 / 16.5
    x[0, 9] = 448.0
    x[0, 10] = torch.arange(32, device="cuda") * 4.0
    x[0, 10, 0, 0] = 127.0                                     # scale 1: whole numbers stay, halves go to even
    x[0, 11] = torch.arange(32, device="cuda") + 0.5
    x[0, 11, 0, 0] = 127.0
    whole = empty_cache(kind, 1, 1, 12, 32)
    starts = torch.zeros(1, dtype=torch.int64, device="cuda")
    ops.kv_write(x, x, starts, *whole)
    codes, scale = quantised(x, kind)
    for c, s in (whole[0::2], whole[1::2]):
        assert np.array_equal(numbers(c)[0, 0], codes[0, :, 0])
        assert np.array_equal(s[0, 0].double().cpu().numpy(), scale[0, :, 0], equal_nan=True)
    got = ops.kv_read(starts, 12, *whole)[0][0, :, 0]
    assert bool(got[1].isnan().all()) and bool(got[2].isnan().all()) and bool((got[[0, 3, 4]] == 0).all())


def test_cache_reads_every_code(native_lib):
    every = torch.arange(256, device="cuda").to(torch.uint8).view(1, 1, 2, 128)
    starts = torch.zeros(1, dtype=torch.int64, device="cuda")
    scale = torch.tensor([0.5, 3.0], device="cuda").view(1, 1, 2)
    got = ops.kv_read(starts, 2, every.view(torch.int8), every.view(torch.int8), scale, scale)[0][0, :, 0]
    assert torch.equal(got, every.view(torch.int8).float()[0, 0] * scale[0, 0][:, None])
    codes = every.view(torch.float8_e4m3fn)
    got = ops.kv_read(starts, 2, codes, codes, scale, scale)[0][0, :, 0]
    want = codes.float()[0, 0] * scale[0, 0][:, None]
    assert torch.equal(got.nan_to_num(7e30), want.nan_to_num(7e30))


def test_cache_rows_outside_and_counts(native_lib):
    k, v = normal(1, 6, 4, 2, 16), normal(2, 6, 4, 2, 16)
    starts = torch.tensor([-2, 3, 5, 2 ** 62, -2 ** 62, 0], device="cuda")
    counts = torch.tensor([4, 4, 4, 4, 4, 2], device="cuda")
    whole = empty_cache("q8", 6, 2, 5, 16)
    ops.kv_write(k, v, starts, *whole, counts=counts)
    rows = {0: {0: 2, 1: 3}, 1: {3: 0, 4: 1}, 5: {0: 0, 1: 1}}       # slot: {cache row: row}
    codes, scale = quantised(k, "q8")
    for b in range(6):
        for at in range(5):
            r = rows.get(b, {}).get(at)
            want = codes[b, r] if r is not None else np.full((2, 16), 7.0)
            assert np.array_equal(numbers(whole[0])[b, :, at], want), (b, at)
            assert float(whole[2][b, 0, at]) == (scale[b, r, 0] if r is not None else 3.0)
    got = ops.kv_read(starts, 4, *whole)[1]
    assert bool((got[0, :2] == 0).all()) and bool((got[1, 2:] == 0).all()) and bool((got[2:5] == 0).all())
    assert torch.equal(got[1, :2], torch.from_numpy(np.multiply(*[a if a.ndim == 4 else a[..., None] for a in quantised(v, "q8")])).float().cuda()[1, :2])
    assert ops.kv_read(starts, 0, *whole)[0].shape == (6, 0, 2, 16)


def test_cache_of_very_many_slots(native_lib):
    slots = 70000
    k = normal(3, slots, 1, 1, 16)
    whole = empty_cache("q8", slots, 1, 2, 16)
    starts = torch.arange(slots, device="cuda") % 2
    ops.kv_write(k, -k, starts, *whole)
    got = ops.kv_read(starts, 1, *whole)
    step = k.abs().amax(-1, keepdim=True) / 127
    # half a step, and the roundings of scale, factor and product: 127 (2 + 1) 2^-24 steps
    assert bool(((got[0] - k).abs() <= 0.50003 * step).all()) and torch.equal(got[1], -got[0])


def test_cache_views(native_lib):
    """Part of a larger cache, heads and rows in another order, entries that are not 16-byte aligned: the same bytes."""
    x = normal(4, 2 * 6 * 3 * 32 + 1)[1:].view(2, 3, 6, 32).transpose(1, 2)
    starts = torch.tensor([1, 0], device="cuda")
    plain, big = empty_cache("e4m3", 2, 3, 8, 32), empty_cache("e4m3", 5, 3, 20, 64)
    part = tuple(t.view(torch.int8)[1:5:2, :, 4:12, 16:48].view(t.dtype) if t.dim() == 4 else t[1:5:2, :, 4:12] for t in big)
    ops.kv_write(x.contiguous(), x.contiguous(), starts, *plain)
    ops.kv_write(x, x, starts, *part)
    for a, b in zip(plain, part):
        assert torch.equal(a.float(), b.float())
    assert bool((big[0].view(torch.int8)[0] == 7).all()) and bool((big[0].view(torch.int8)[..., :16] == 7).all())
    assert all(torch.equal(a, b) for a, b in zip(ops.kv_read(starts, 6, *plain), ops.kv_read(starts, 6, *part)))


# ---- attention --------------------------------------------------------------------------------------------------------
def make_cache(kind, seed, slots, heads, cap, d):
    """(arguments, keys, values): what the operator takes, and what it stands for in 64 bits."""
    k, v = normal(seed, slots, heads, cap, d), normal(seed + 1, slots, heads, cap, d) + 0.3
    if kind in TYPES:
        k, v = k.to(TYPES[kind]), v.to(TYPES[kind])
        return (k, v, None, None), k.double(), v.double()
    whole = empty_cache(kind, slots, heads, cap, d)
    ops.kv_write(k.transpose(1, 2), v.transpose(1, 2), torch.zeros(slots, dtype=torch.int64, device="cuda"), *whole)
    codes = [c.float().double() for c in whole[:2]]
    return whole, codes[0] * whole[2][..., None].double(), codes[1] * whole[3][..., None].double()


def attended(q, k, v, lengths, mask, scale):
    """(result, bound) of every row."""
    slots, rows, heads, d = q.shape
    cap, group = k.shape[2], heads // k.shape[1]
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b in range(slots):
        n = int(lengths[b])
        if n < 0:
            continue
        n = min(n, cap)
        total = min(n + rows, cap)
        seen = torch.cat([torch.ones(rows, n, dtype=torch.bool, device="cuda"), mask[b][:, :total - n]], 1)
        for h in range(heads):
            keys, values = k[b, h // group, :total], v[b, h // group, :total]
            scores = (q[b, :, h].double() @ keys.T * scale).masked_fill(~seen, -math.inf)
            top = scores.amax(-1, keepdim=True)
            w = torch.exp(scores - torch.where(top == -math.inf, 0.0, top)).masked_fill(~seen, 0)
            w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
            out[b, :, h] = w @ torch.where(seen.any(0)[:, None], values, 0.0)
            # a score: up to 24 accumulations, the query's terms and three f32 operations, relative to the sum of magnitudes; a
            # weight: twice that, the exponential and its operand's rounding; then values times weights' errors
            size = ((q[b, :, h].double().abs() @ keys.abs().T) * scale).masked_fill(~seen, 0).amax(-1, keepdim=True)
            weight = 2 * (24 * 2.0 ** -23 + 2.0 ** -20) * size + 2.0 ** -18
            if q.dtype != torch.float32:
                weight = weight + 2.0 ** -12        # weights of one f16 term, or two bf16 ones
            # and an absolute part: a weight enters as f16 times at least 2^13 / (the largest value's scale). f16 has steps of 2^-24, so
            # its last term is off by up to 2^-25 there, which is 2^-38 of the largest value for every key
            steps = total * 2.0 ** -38 * torch.where(seen.any(0)[:, None], values.abs(), 0.0).amax()
            bound[b, :, h] = weight * (w @ torch.where(seen.any(0)[:, None], values.abs(), 0.0)) + steps
    return out, bound + half(q.dtype) * (out.abs() + bound)


def tree_mask(seed, slots, rows):
    g = torch.Generator().manual_seed(seed)
    mask = torch.rand(slots, rows, rows, generator=g) < 0.4
    mask[:, rows // 2] = False                       # a row that sees none of the tree
    return mask.cuda()


ATTEND = [  # slots, rows, heads, kv heads, d, lengths, capacity
    (1, 1, 1, 1, 16, [0], 1), (1, 1, 8, 8, 128, [1], 2), (2, 1, 16, 2, 128, [300, 17], 400), (1, 5, 16, 8, 128, [600], 605),
    (3, 3, 6, 2, 64, [0, 31, 32], 64), (2, 16, 4, 4, 128, [15, 16], 64), (2, 13, 32, 8, 128, [1000, 77], 1200),
    (1, 33, 5, 5, 80, [255], 300), (1, 33, 4, 2, 96, [1], 34), (2, 64, 8, 2, 128, [513, 2], 600), (1, 70, 6, 1, 48, [129], 200),
    (1, 129, 2, 1, 128, [65], 194), (5, 2, 4, 1, 112, [-1, 3, 0, -5, 40], 50), (1, 1, 40, 1, 128, [5000], 5001),
    (1, 1, 8, 1, 128, [20000], 20001), (1, 4, 4, 1, 64, [9000], 9004), (40, 1, 16, 16, 64, list(range(0, 400, 10)), 420),
    # clusters of sizes that are no power of two, and of sixteen blocks for many rows
    (1, 20, 3, 1, 64, [5000], 5020), (1, 17, 10, 10, 128, [3000], 3017), (2, 30, 30, 5, 128, [4100, 0], 4140),
    (2, 1, 8, 8, 128, [4000, 7], 4001), (1, 3, 68, 17, 64, [3000], 3003),
]


@pytest.mark.parametrize("cache", ["bf16", "f16", "q8", "e4m3"])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("slots,rows,heads,kv,d,lengths,cap", ATTEND)
def test_tree_attention(native_lib, cache, kind, slots, rows, heads, kv, d, lengths, cap):
    args, k, v = make_cache(cache, 21, slots, kv, cap, d)
    q = (1.5 * normal(5, slots, rows, heads, d)).to(TYPES[kind])
    mask = tree_mask(rows, slots, rows)
    n = torch.tensor(lengths, device="cuda")
    got = ops.tree_attention(q, args[0], args[1], n, mask, args[2], args[3])
    want, bound = attended(q, k, v, lengths, mask, d ** -0.5)
    assert got.dtype == q.dtype and bool(((got.double() - want).abs() <= bound).all()), float((got.double() - want).abs().max())
    for b in range(slots):                               # nothing to see: exactly zero
        empty = ~mask[b].any(-1) if lengths[b] == 0 else torch.full((rows,), lengths[b] < 0, device="cuda")
        assert bool((got[b][empty] == 0).all())
    again = ops.tree_attention(q, args[0], args[1], n, mask, args[2], args[3])
    assert torch.equal(got, again)


@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_tree_attention_without_a_mask_is_a_chain(native_lib, cache):
    args, k, v = make_cache(cache, 3, 2, 2, 90, 64)
    q, n = normal(1, 2, 7, 4, 64), torch.tensor([80, 11], device="cuda")
    chain = torch.ones(7, 7, device="cuda").tril().bool()
    got = ops.tree_attention(q, args[0], args[1], n, None, args[2], args[3], scale=0.3)
    assert torch.equal(got, ops.tree_attention(q, args[0], args[1], n, chain, args[2], args[3], scale=0.3))
    want, bound = attended(q, k, v, [80, 11], chain.expand(2, 7, 7), 0.3)
    assert bool(((got.double() - want).abs() <= bound).all())


def test_tree_attention_agrees_with_attention(native_lib):
    """A chain over a bf16 cache is what `ops.attention` computes."""
    args, _, _ = make_cache("bf16", 9, 1, 8, 700, 128)
    q = normal(2, 1, 5, 16, 128)
    got = ops.tree_attention(q, args[0], args[1], torch.tensor([600], device="cuda"))
    want = ops.attention(q[0], args[0][0], args[1][0], 600).view(5, 16, 128)
    assert float((got[0] - want).abs().max()) < 2e-5


def test_tree_attention_keys_end_at_the_capacity(native_lib):
    args, k, v = make_cache("q8", 5, 2, 1, 40, 64)
    q, mask = normal(3, 2, 9, 2, 64), tree_mask(1, 2, 9)
    n = torch.tensor([36, 1000], device="cuda")
    want, bound = attended(q, k, v, [36, 40], mask, 0.125)
    got = ops.tree_attention(q, args[0], args[1], n, mask, args[2], args[3])
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("cache", ["bf16", "f16"])
@pytest.mark.parametrize("rows,heads", [(5, 4), (40, 4), (70, 2)])
def test_values_that_are_not_finite_reach_those_that_see_them(native_lib, cache, rows, heads):
    args, k, v = make_cache(cache, 31, 1, 2, 300, 128)
    q = normal(4, 1, rows, heads, 128)
    mask = torch.zeros(1, rows, rows, dtype=torch.bool, device="cuda")
    mask[0, :, 0] = True
    mask[0, 3, 2] = mask[0, 1, 1] = mask[0, 4, 3] = True
    base = 200
    args[1][0, 0, base + 2, 5] = math.inf
    args[1][0, 0, base + 1, 9] = math.nan
    args[0][0, 0, base + 4] = math.nan                       # a key that nobody sees
    args[0][0, 0, base + rows:] = math.nan                   # behind the tree
    args[1][0, 1, base + rows:] = -math.inf
    args[1][0, 0, base + 3, 7], args[1][0, 1, 17, 3] = -math.inf, math.inf
    n = torch.tensor([base], device="cuda")
    got = ops.tree_attention(q, args[0], args[1], n, mask)[0].double()
    clean_k, clean_v = args[0].double().nan_to_num(0, 0, 0), args[1].double().nan_to_num(0, 0, 0)
    want, bound = attended(q, clean_k, clean_v, [base], mask, 128 ** -0.5)
    want, bound = want[0], bound[0]
    group = heads // 2
    want[3, :group, 5], want[1, :group, 9], want[4, :group, 7] = math.inf, math.nan, -math.inf
    want[:, group:, 3] = math.inf                            # in front of the tree: everybody sees it
    fine = want.isfinite()
    assert bool(((got - want).abs() <= bound)[fine].all())
    assert torch.equal(got[~fine].nan_to_num(7e300), want[~fine].nan_to_num(7e300))


def test_codes_that_are_not_numbers_reach_those_that_see_them(native_lib):
    """e4m3's NaN codes, which no write makes, in rows that nobody or not everybody sees."""
    args, k, v = make_cache("e4m3", 37, 1, 1, 90, 128)
    codes = args[1].view(torch.uint8)
    codes[0, 0, 50 + 2, 77], codes[0, 0, 60:] = 0xff, 0x7f
    args[0].view(torch.uint8)[0, 0, 56:] = 0x7f
    for rows, heads in ((5, 1), (5, 3), (8, 3)):
        q, mask = normal(4, 1, rows, heads, 128), torch.zeros(1, rows, rows, dtype=torch.bool, device="cuda")
        mask[0, 1, 2] = mask[0, 3, 3] = True
        got = ops.tree_attention(q, args[0], args[1], torch.tensor([50], device="cuda"), mask, args[2], args[3])
        want, bound = attended(q, k, v.nan_to_num(0), [50], mask, 128 ** -0.5)
        nan = torch.zeros_like(want, dtype=torch.bool)
        nan[0, 1, :, 77] = True
        assert torch.equal(got.isnan(), nan) and bool(((got.double() - want).abs() <= bound)[~nan].all())


@pytest.mark.parametrize("cache", ["bf16", "q8"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [3, 12, 40])
def test_queries_that_are_not_finite_spoil_their_own_rows_only(native_lib, cache, kind, rows):
    """As a padded batch may hold them."""
    args, k, v = make_cache(cache, 39, 2, 1, 500, 64)
    q, mask = normal(4, 2, rows, 2, 64).to(TYPES[kind]), tree_mask(3, 2, rows)
    clean = q.clone()
    q[0, rows - 1], q[1, 1, 0, 5], q[1, 2, 1, 9] = math.nan, math.inf, -math.inf
    spoilt = ~q.isfinite().all(-1)
    n = torch.tensor([400, 333], device="cuda")
    got = ops.tree_attention(q, args[0], args[1], n, mask, args[2], args[3])
    want, bound = attended(torch.where(spoilt[..., None], 0.0, q.float()).to(q.dtype), k, v, [400, 333], mask, 0.125)
    assert bool(((got.double() - want).abs() <= bound)[~spoilt].all()) and bool(got[spoilt].isnan().all())
    assert torch.equal(got[~spoilt], ops.tree_attention(clean, args[0], args[1], n, mask, args[2], args[3])[~spoilt])


@pytest.mark.parametrize("cache", ["q8", "e4m3"])
def test_a_row_of_an_8_bit_cache_that_is_not_a_number(native_lib, cache):
    args, k, v = make_cache(cache, 33, 1, 1, 100, 64)
    q, mask = normal(4, 1, 4, 2, 64), torch.eye(4, dtype=torch.bool, device="cuda")[None]
    args[2][0, 0, 52] = math.nan                             # the key of row 2
    args[3][0, 0, 53] = math.nan                             # the value of row 3
    args[2][0, 0, 54:], args[3][0, 0, 54:] = math.nan, math.inf
    got = ops.tree_attention(q, args[0], args[1], torch.tensor([50], device="cuda"), mask, args[2], args[3])
    want, bound = attended(q, k, v, [50], mask, 0.125)
    assert bool(((got.double() - want).abs() <= bound)[0, :2].all()) and bool(got[0, 2:].isnan().all())


def test_extreme_queries_and_scales(native_lib):
    """Large and small queries meet scales that keep the scores moderate: rows are scaled on their own."""
    args, k, v = make_cache("q8", 35, 1, 1, 64, 128)
    q = normal(4, 1, 4, 2, 128)
    mask, n = torch.ones(1, 4, 4, dtype=torch.bool, device="cuda"), torch.tensor([60], device="cuda")
    for size in (1e-30, 1e-6, 1e6, 1e25):
        got = ops.tree_attention(q * size, args[0], args[1], n, mask, args[2], args[3], scale=0.09 / size)
        want, bound = attended(q * size, k, v, [60], mask, 0.09 / size)
        assert bool(((got.double() - want).abs() <= bound).all()), size
        got = ops.tree_attention(q, args[0], args[1], n, mask, args[2] * size, args[3] * size, scale=0.09 / size)
        want, bound = attended(q, k * size, v * size, [60], mask, 0.09 / size)
        # the scales times the size are rounded once more than in `attended`: 2^-24 of a score and of a value
        bound = bound * 1.1 + 2.0 ** -23 * want.abs()
        assert bool(((got.double() - want).abs() <= bound).all()), size
    # weights far below one another, and values whose scales differ by ten orders
    args[3][0, 0, ::3] *= 1e-10
    want, bound = attended(8 * q, k, args[1].double() * args[3][..., None].double(), [60], mask, 1.0)
    got = ops.tree_attention(8 * q, args[0], args[1], n, mask, args[2], args[3], scale=1.0)
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_tree_attention_views_and_far_offsets(native_lib, cache):
    """Slots and heads more than 2^32 bytes apart, queries and masks out of larger tensors."""
    d, cap, size = 64, 70, 2 if cache == "bf16" else 1
    args, k, v = make_cache(cache, 41, 2, 2, cap, d)
    q, mask = normal(6, 2, 6, 8, 2 * d)[:, :, 2:6, d:], tree_mask(7, 2, 12)[:, 3:9, 5:11]
    big = torch.empty((5 << 30) + 4 * cap * d, dtype=torch.int8, device="cuda")
    far = [torch.as_strided(big.view(args[0].dtype), (2, 2, cap, d), ((4 << 30) // size, (1 << 29) // size, d, 1), i * cap * d) for i in (0, 1)]
    for to, of in zip(far, args[:2]):
        to.view(torch.int8).copy_(of.view(torch.int8))
    n = torch.tensor([64, 50], device="cuda")
    got = ops.tree_attention(q, far[0], far[1], n, mask, args[2], args[3])
    assert torch.equal(got, ops.tree_attention(q.contiguous(), args[0], args[1], n, mask.contiguous(), args[2], args[3]))
    want, bound = attended(q, k, v, [64, 50], mask, 0.125)
    assert bool(((got.double() - want).abs() <= bound).all())


# ---- verification -----------------------------------------------------------------------------------------------------
def verified(tokens, parents, target, u, draft):
    """The definition, one sequence after the other, with sums in 64 bits."""
    counts, paths, drawn = [], [], []
    for b in range(target.shape[0]):
        path, z, gone = [0], 1.0, 0
        p = target[b].double().cpu().numpy()
        q = None if draft is None else draft[b].double().cpu().numpy()
        r = p[0].copy()
        for i in range(1, target.shape[1]):
            if int(parents[b, i]) != path[-1]:
                continue
            x = int(tokens[b, i])
            inside = 0 <= x < len(r)
            chance = (1.0 if q is None else q[path[-1]][x]) if inside else 0.0
            if inside and float(u[b, i]) * chance * z < r[x]:
                path.append(i)
                r, z = p[i].copy(), 1.0
            elif q is None:
                if inside:
                    z -= r[x]
                    r[x] = 0
            else:
                r = np.maximum((r / z if z > 0 else 0 * r) - q[path[-1]], 0)
                z = r.sum()
        if r.sum() == 0:
            r = p[path[-1]]
        total = r.sum()
        if not (np.isfinite(total) and total > 0):
            drawn.append(-1)
        else:
            sums = np.cumsum(r)
            beyond = np.nonzero(sums > float(u[b, 0]) * sums[-1])[0]
            drawn.append(int(beyond[0]) if len(beyond) else int(np.nonzero(r)[0][-1]))
        counts.append(len(path) - 1)
        paths.append(path + [-1] * (target.shape[1] - len(path)))
    return counts, paths, drawn


def check_verified(tokens, parents, target, u, draft=None):
    got = ops.verify_draft(tokens, parents, target, u, draft)
    whole = parents if parents.dim() == 2 else parents.expand(target.shape[0], -1)
    want = verified(tokens, whole, target, u, draft)
    for g, w, name in zip(got, want, ("accepted", "path", "next")):
        assert g.dtype == torch.int64 and g.tolist() == w, name
    return got


def drafted(seed, slots, nodes, vocab, kind, tree, sharp=2.0):
    g = torch.Generator("cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    logits = sharp * torch.randn(slots, nodes, vocab, generator=g, device="cuda")
    target = torch.softmax(logits, -1).to(TYPES[kind])
    draft = torch.softmax(0.8 * logits + 0.5 * torch.randn(slots, nodes, vocab, generator=g, device="cuda"), -1).to(TYPES[kind])
    parents = np.arange(nodes)[None].repeat(slots, 0) - 1
    if tree:
        parents = np.maximum(parents - rng.integers(0, 4, size=parents.shape), 0)
        parents[:, 0] = -1
    parents = torch.from_numpy(parents).cuda()
    up = draft.float()[torch.arange(slots, device="cuda")[:, None], parents.clamp(min=0)]
    tokens = torch.multinomial(up.view(-1, vocab), 1, generator=g).view(slots, nodes)
    return tokens, parents, target, torch.rand(slots, nodes, generator=g, device="cuda"), draft


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("slots,nodes,vocab,kind", [(1, 1, 1, "f32"), (3, 2, 2, "f32"), (40, 9, 33, "f32"), (7, 5, 1000, "bf16"), (5, 30, 4097, "f16"),
                                                    (300, 4, 257, "f32"), (1, 5, 151936, "f32"), (20, 6, 50001, "bf16"),
                                                    (33, 4, 20001, "f32"), (45, 3, 20001, "bf16"), (63, 3, 20003, "f16")])
def test_verify_draft(native_lib, slots, nodes, vocab, kind, with_draft, tree):
    for seed in (1, 2):
        tokens, parents, target, u, draft = drafted(seed, slots, nodes, vocab, kind, tree)
        check_verified(tokens, parents, target, u, draft if with_draft else None)


def test_verify_edges(native_lib):
    tokens, parents, target, u, draft = drafted(5, 8, 6, 500, "f32", True)
    for edge in (0.0, float(np.nextafter(np.float32(1), np.float32(0))), 1.0):       # 1 is outside the range: the last entry left
        check_verified(tokens, parents, target, torch.full_like(u, edge), draft)
        check_verified(tokens, parents, target, torch.full_like(u, edge))
    # the target is the draft: after a refusal nothing is left, and the row itself is drawn from
    same = u.clone()
    same[:, 1:] = 1.0
    check_verified(tokens, parents, target, same, target)
    # tokens outside the vocabulary and the same token twice
    wrong = tokens.clone()
    wrong[:4, 1:3], wrong[4:, 1:] = torch.tensor([-1, 500], device="cuda"), 7
    check_verified(wrong, parents, target, u, draft)
    check_verified(wrong, parents, target, u)
    # nodes that are not there, and parents that make no sense
    holes = parents.clone()
    holes[:3, 2:], holes[3, 1:] = -1, torch.tensor([5, 9, -7, 3, 2 ** 40], device="cuda")
    check_verified(tokens, holes, target, u, draft)
    # one tree for all; all mass on one token that is refused; rows without a sum
    check_verified(tokens, parents[0], target, u, draft)
    point = torch.zeros_like(target)
    point[..., 7] = 1.0
    check_verified(wrong, parents, point, torch.full_like(u, 0.999), point)
    check_verified(wrong, parents, point, u)
    bad = target.clone()
    bad[0], bad[1, :, 3], bad[2, :, 5], bad[3] = 0.0, math.nan, math.inf, 0.0
    check_verified(tokens, parents, bad, u, draft)
    check_verified(tokens, parents, bad, u)


def test_verify_views_and_many_nodes(native_lib):
    tokens, parents, target, u, draft = drafted(6, 4, 7, 301, "f32", True)
    wide = torch.zeros(4, 9, 2, 400, device="cuda")
    wide[:, 1:8, 0, 50:351], wide[:, 1:8, 1, 50:351] = target, draft
    check_verified(tokens.t().contiguous().t(), parents.to(torch.int32), wide[:, 1:8, 0, 50:351], u, wide[:, 1:8, 1, 50:351])
    tokens, parents, target, u, draft = drafted(7, 2, 1024, 40, "f16", True)
    check_verified(tokens, parents, target, u, draft)
    check_verified(tokens, parents, target, u)


def test_the_target_distribution_is_kept(native_lib):
    """One drafted level of three children and many random numbers: the first token behind the text is distributed as the target's
    row. 2^15 trials of six tokens: a frequency is within six standard deviations, of at most 0.5 / sqrt(trials)."""
    trials, vocab = 1 << 15, 6
    g = torch.Generator("cuda").manual_seed(11)
    p = torch.tensor([0.35, 0.3, 0.2, 0.1, 0.05, 0.0], device="cuda")
    q = torch.tensor([0.05, 0.3, 0.1, 0.2, 0.25, 0.1], device="cuda")
    target, draft = p.expand(trials, 4, vocab), q.expand(trials, 4, vocab)
    parents = torch.tensor([-1, 0, 0, 0], device="cuda")
    u = torch.rand(trials, 4, generator=g, device="cuda")
    for chosen in (False, True):
        tokens = torch.tensor([0, 1, 4, 0], device="cuda").expand(trials, 4) if chosen else \
            torch.multinomial(q, 4 * trials, replacement=True, generator=g).view(trials, 4)
        count, path, token = ops.verify_draft(tokens, parents, target, u, None if chosen else draft)
        first = torch.where(count > 0, tokens.gather(1, path[:, 1:2].clamp(min=0))[:, 0], token)
        got = torch.bincount(first, minlength=vocab).double() / trials
        assert float((got - p).abs().max()) < 6 * 0.5 / math.sqrt(trials), (chosen, got)


# ---- together, and how they are called --------------------------------------------------------------------------------
def step_inputs(seed, slots=3, rows=6, heads=8, kv=2, d=64, vocab=997):
    qkv = normal(seed, slots, rows, heads + 2 * kv, d)
    tokens, parents, target, u, draft = drafted(seed, slots, rows, vocab, "f32", True)
    depth, mask = torch.zeros_like(parents), torch.zeros(slots, rows, rows, dtype=torch.bool, device="cuda")
    for b in range(slots):
        for i in range(rows):
            if i:
                depth[b, i] = depth[b, parents[b, i]] + 1
                mask[b, i] = mask[b, parents[b, i]]
            mask[b, i, i] = True
    return qkv, tokens, parents, target, u, draft, depth, mask


@pytest.mark.parametrize("kind", ["q8", "e4m3"])
def test_a_whole_step(native_lib, kind):
    """Rotate at the nodes' depths, write behind the cache, attend, verify, and write the rows that stand in their order."""
    slots, rows, heads, kv, d, cap = 3, 6, 8, 2, 64, 120
    qkv, tokens, parents, target, u, draft, depth, mask = step_inputs(1)
    whole = empty_cache(kind, slots, kv, cap, d)
    lengths = torch.tensor([100, 37, 0], device="cuda")
    past = normal(2, slots, 100, 2 * kv, d)
    ops.kv_write(past[:, :, :kv], past[:, :, kv:], torch.zeros_like(lengths), *whole, counts=lengths)
    f, _ = ops.rotary_frequencies(d)
    x = qkv.clone()
    ops.rotary(x[:, :, :heads + kv], lengths[:, None] + depth, f, out=x[:, :, :heads + kv])
    ops.kv_write(x[:, :, heads:heads + kv], x[:, :, heads + kv:], lengths, *whole)
    out = ops.tree_attention(x[:, :, :heads], whole[0], whole[1], lengths, mask, *whole[2:])
    count, path, token = ops.verify_draft(tokens, parents, target, u, draft)
    # the path's rows move to the front of the tree's place: kept rows of k and v, the others left out
    kept = x[torch.arange(slots, device="cuda")[:, None], path.clamp(min=0)]
    ops.kv_write(kept[:, :, heads:heads + kv], kept[:, :, heads + kv:], lengths, *whole, counts=count + 1)

    turned, _ = rotated(qkv[:, :, :heads + kv], (lengths[:, None] + depth).double()[..., None] * f.cuda(), d, "half", 1.0)
    assert float((x[:, :, :heads + kv].double() - turned).abs().max()) < 1e-5
    assert torch.equal(x[:, :, heads + kv:], qkv[:, :, heads + kv:])
    rows_of = [np.multiply(c, s[..., None]) for c, s in (quantised(t, kind) for t in (past[:, :, :kv], past[:, :, kv:], x[:, :, heads:heads + kv], x[:, :, heads + kv:]))]
    k, v = (torch.zeros(slots, kv, cap, d, dtype=torch.float64, device="cuda") for _ in "kv")
    for b in range(slots):
        n = int(lengths[b])
        for to, old, new in ((k, rows_of[0], rows_of[2]), (v, rows_of[1], rows_of[3])):
            to[b, :, :n] = torch.from_numpy(old[b, :n]).cuda().transpose(0, 1)
            to[b, :, n:n + rows] = torch.from_numpy(new[b]).cuda().transpose(0, 1)
    want, bound = attended(x[:, :, :heads], k, v, lengths.tolist(), mask, d ** -0.5)
    assert bool(((out.double() - want).abs() <= bound).all())
    assert [count.tolist(), path.tolist(), token.tolist()] == list(verified(tokens, parents, target, u, draft))
    got = ops.kv_read(lengths, rows, *whole)[0].double().cpu().numpy()
    for b in range(slots):
        for i in range(rows):
            node = int(path[b, i]) if i <= int(count[b]) else i        # behind the path: as the tree left them
            assert np.array_equal(got[b, i].astype(np.float32), rows_of[2][b, node].astype(np.float32))


def whole_step(x, whole, lengths, positions, mask, tokens, parents, target, u, draft, f, heads=8, kv=2):
    ops.rotary(x[:, :, :heads + kv], positions, f, out=x[:, :, :heads + kv])
    ops.kv_write(x[:, :, heads:heads + kv], x[:, :, heads + kv:], lengths, *whole)
    out = ops.tree_attention(x[:, :, :heads], whole[0], whole[1], lengths, mask, *whole[2:])
    return (out, *ops.kv_read(lengths, x.shape[1], *whole), *ops.verify_draft(tokens, parents, target, u, draft))


def test_captured_replayed_and_on_other_streams(native_lib):
    """A step in a graph, replayed on new contents; two graphs and an eager step on streams of their own at the same time."""
    f, _ = ops.rotary_frequencies(64)
    lengths = torch.tensor([90, 37, 0], device="cuda")

    def make(seed):
        qkv, tokens, parents, target, u, draft, depth, mask = step_inputs(seed)
        return [qkv, empty_cache("q8", 3, 2, 120, 64), lengths.clone(), lengths[:, None] + depth, mask, tokens, parents, target, u, draft, f]

    def copied(s):
        return [t.clone() if isinstance(t, torch.Tensor) and t.is_cuda else tuple(c.clone() for c in t) if isinstance(t, tuple) else t for t in s]

    want = {seed: [t.clone() for t in whole_step(*copied(make(seed)))] for seed in (1, 2, 3)}
    captured = []
    for seed in (1, 2):
        state = make(seed)
        fresh = copied(state)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            whole_step(*copied(state))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = whole_step(*state)
        captured.append((graph, state, fresh, out, seed))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for (graph, state, fresh, out, seed), stream in zip(captured, streams):
            with torch.cuda.stream(stream):
                state[0].copy_(fresh[0])
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = whole_step(*copied(make(3)))
    torch.cuda.synchronize()
    for (_, _, _, out, seed) in captured:
        assert all(torch.equal(a, b) for a, b in zip(out, want[seed]))
    assert all(torch.equal(a, b) for a, b in zip(eager, want[3]))
    # replayed on other contents
    graph, state, fresh, out, _ = captured[0]
    for to, of in zip(state, make(2)):
        if isinstance(to, tuple):
            for a, b in zip(to, of):
                a.view(torch.uint8).copy_(b.view(torch.uint8))
        elif to.is_cuda:
            to.copy_(of)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want[2]))


def test_tensors_on_different_devices_are_refused(native_lib):
    with pytest.raises(ValueError, match="different devices"):
        ops.rotary(normal(1, 3, 2, 8), torch.arange(3), torch.ones(4, dtype=torch.float64))
