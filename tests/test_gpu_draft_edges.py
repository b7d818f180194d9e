"""The operators of speculative decoding at the ends of their ranges. Bounds as in `test_gpu_draft`, with absolute parts that
count only the keys that a row sees.
"""
import math
import os
import subprocess
import sys
import textwrap
from fractions import Fraction

import pytest
import torch

from dyninfer_b200 import ops
from test_gpu_draft import TYPES, half, make_cache, normal

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def attended_by_row(q, k, v, n, mask, scale):
    """(result, bound) of q [rows, heads, d] over one sequence's k and v [kv heads, keys, d] in 64 bits."""
    rows, heads, d = q.shape
    group = heads // k.shape[0]
    seen = torch.cat([torch.ones(rows, n, dtype=torch.bool, device="cuda"), mask], 1)
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for h in range(heads):
        keys, values = k[h // group, :n + rows], torch.where(seen[..., None], v[h // group, :n + rows], 0.0)     # [row, key, d]
        products = torch.where(seen[..., None], q[:, h].double()[:, None] * keys * scale, 0.0)
        scores = products.sum(-1).masked_fill(~seen, -math.inf)
        top = scores.amax(-1, keepdim=True)
        w = torch.exp(scores - torch.where(top == -math.inf, 0.0, top)).masked_fill(~seen, 0)
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        out[:, h] = torch.where(w[..., None] > 0, w[..., None] * values, 0.0).sum(1)
        # a score: up to 24 accumulations, the query's terms and three f32 operations, relative to the sum of magnitudes; a weight:
        # twice that, the exponential, and its rounding as an operand: one f16 term for bf16 queries (two for the others)
        size = torch.where(products.isfinite(), products.abs(), 0.0).sum(-1).amax(-1, keepdim=True)
        weight = 2 * (24 * 2.0 ** -23 + 2.0 ** -20) * size + 2.0 ** -18 + (2.0 ** -11 if q.dtype == torch.bfloat16 else 0)
        # a weight's last f16 term is off by up to 2^-25, in units of 2^-13 (f32 queries) or 2^-5 of the largest value scale that
        # the row sees
        steps = (n + rows) * 2.0 ** (-38 if q.dtype == torch.float32 else -30) * values.abs().amax((1, 2))[:, None]
        bound[:, h] = weight * torch.where(w[..., None] > 0, w[..., None] * values.abs(), 0.0).sum(1) + steps
    # the result's rounding; f16 has steps of 2^-24 below 2^-14
    return out, bound + half(q.dtype) * (out.abs() + bound) + (2.0 ** -25 if q.dtype == torch.float16 else 0)


@pytest.mark.parametrize("cache", ["q8", "e4m3"])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,n", [(4, 50), (8, 50), (20, 50), (4, 500), (8, 500), (64, 500), (20, 0)])
def test_value_scales_of_keys_that_are_not_seen(native_lib, cache, kind, rows, n):
    """Two query heads share a kv head: up to 8 rows, up to 16, and more. A node that nobody sees, and one that a single row does."""
    args, k, v = make_cache(cache, 43, 1, 2, n + rows + 3, 128)
    q = normal(8, 1, rows, 4, 128).to(TYPES[kind])
    mask = torch.rand(rows, rows, device="cuda", generator=torch.Generator("cuda").manual_seed(rows)) < 0.5
    hidden, alone, seer = rows // 2, rows - 1, 1
    mask[:, hidden] = mask[:, alone] = False
    mask[seer, alone] = True
    codes = args[1].float().double()
    length = torch.tensor([n], device="cuda")
    clean = None
    for size in (1.0, 2.0 ** 25, 2.0 ** 40, 1e10, 1e30, math.inf):
        args[3][0, :, n + hidden] = size
        args[3][0, :, n + alone] = min(size, 1e10)
        got = ops.tree_attention(q, args[0], args[1], length, mask, args[2], args[3])[0]
        v = codes * args[3][..., None].double()
        want, bound = attended_by_row(q[0], k[0], v[0], n, mask, 128 ** -0.5)
        near = ((got.double() - want).abs() <= bound) | (got == want.to(got.dtype))       # the latter: infinity beyond f16's range
        assert bool(near.all()), (size, float((got.double() - want)[~near].abs().max()))
        # and those that see neither are what they are beside a small scale
        rest = torch.arange(rows, device="cuda") != seer
        clean = got if clean is None else clean
        assert torch.equal(got[rest], clean[rest]), size


def test_a_form_is_captured_that_was_not_called_before(native_lib):
    """One call of the operator has been made, with few rows; the captured one has many. In a process of its own, where no
    other operator has set anything up."""
    text = textwrap.dedent("""
        import torch
        from dyninfer_b200 import ops
        q = torch.randn(1, 40, 4, 64, device="cuda")
        k, v = (torch.randn(1, 2, 400, 64, device="cuda").bfloat16() for _ in range(2))
        n = torch.tensor([300], device="cuda")
        ops.tree_attention(q[:, :2].contiguous(), k, v, n)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.tree_attention(q, k, v, n)
        graph.replay()
        want = ops.tree_attention(q, k, v, n)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        print("same")
    """)
    done = subprocess.run([sys.executable, "-c", text], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert done.returncode == 0 and done.stdout.split() == ["same"], done.stderr[-2000:]


def test_rotary_fractions_are_rounded(native_lib):
    """At 2^60 a fraction of a turn that is off by 2^-65 moves the angle by 2^-5 turns, one off by 2^-64 by 2^-4."""
    f, _ = ops.rotary_frequencies(128, 1e4)
    pi = Fraction(3141592653589793238462643383279502884197169399, 10 ** 45)
    position = 2 ** 60
    want = [float((Fraction(position) * Fraction(float(w)) / (2 * pi)) % 1) for w in f]
    x = torch.cat([torch.ones(1, 1, 64, device="cuda"), torch.zeros(1, 1, 64, device="cuda")], -1)
    got = ops.rotary(x, torch.tensor([position], device="cuda"), f)[0, 0].double().cpu()
    turns = torch.atan2(got[64:], got[:64]) / (2 * math.pi)
    off = (turns - torch.tensor(want, dtype=torch.float64)).remainder(1)
    # the fraction's rounding to 2^-64; one over 2 pi, and the product with it, both below a quarter, rounded to 64 bits: 2^-67 each.
    # Then cosine and sine in f32, 2^-22 radians at most
    assert float(torch.minimum(off, 1 - off).max()) <= position * (2.0 ** -65 + 2 * 2.0 ** -67) + 2.0 ** -22


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 8, 20])
@pytest.mark.parametrize("cache", ["q8", "e4m3"])
def test_value_scales_near_the_end_of_f32(native_lib, cache, kind, rows):
    """Values up to 2^126; a row sees four keys, so that their sum is a number as well."""
    args, k, v = make_cache(cache, 44, 1, 1, 3 + rows, 64)
    args[3].mul_(2.0 ** 124)
    v = v * 2.0 ** 124
    q, mask = normal(9, 1, rows, 2, 64).to(TYPES[kind]), torch.eye(rows, dtype=torch.bool, device="cuda")
    got = ops.tree_attention(q, args[0], args[1], torch.tensor([3], device="cuda"), mask, args[2], args[3])[0]
    want, bound = attended_by_row(q[0], k[0], v[0], 3, mask, 0.125)
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("rows", [2, 8, 20])
def test_queries_near_the_end_of_f32(native_lib, rows):
    args, k, v = make_cache("q8", 45, 1, 1, 60 + rows, 128)
    args[2].mul_(2.0 ** -110)
    q, mask = normal(9, 1, rows, 2, 128), torch.eye(rows, dtype=torch.bool, device="cuda")
    q *= 3.39e38 / q.abs().amax(-1, keepdim=True)
    k, scale = k * 2.0 ** -110, 2.0 ** -17
    got = ops.tree_attention(q, args[0], args[1], torch.tensor([60], device="cuda"), mask, args[2], args[3], scale=scale)[0]
    want, bound = attended_by_row(q[0], k[0], v[0], 60, mask, scale)
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("cache", ["bf16", "f16", "q8", "e4m3"])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [3, 8, 20])
def test_infinite_queries_whose_scores_are_all_minus_infinity(native_lib, cache, kind, rows):
    """No weights come of them: such a row is not a number, wherever it sees a key, and zeros where it sees none."""
    args, k, v = make_cache(cache, 47, 1, 1, 1 + rows, 64)
    q = normal(9, 1, rows, 2, 64).to(TYPES[kind])
    first = int((k[0, 0, 0] < 0).nonzero()[0])               # a dimension in which the only key is below zero
    q[0, 1, :, first] = math.inf
    mask = torch.zeros(rows, rows, dtype=torch.bool, device="cuda")
    want, bound = attended_by_row(q[0].nan_to_num(posinf=0.0), k[0], v[0], 1, mask, 0.125)
    got = ops.tree_attention(q, args[0], args[1], torch.tensor([1], device="cuda"), mask, args[2], args[3])[0]
    rest = torch.arange(rows, device="cuda") != 1
    assert bool(got[1].isnan().all()) and bool(((got.double() - want).abs() <= bound)[rest].all())
    got = ops.tree_attention(q, args[0], args[1], torch.tensor([0], device="cuda"), mask, args[2], args[3])
    assert bool((got == 0).all())


@pytest.mark.parametrize("cache", ["bf16", "f16"])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [3, 8, 20])
def test_infinite_keys_that_are_seen(native_lib, cache, kind, rows):
    """A score of minus infinity is a weight of zero; one of plus infinity, or an infinity against a zero, spoils the row."""
    args, k, v = make_cache(cache, 46, 1, 1, 90 + rows, 64)
    q = normal(9, 1, rows, 2, 64).to(TYPES[kind])
    q[0, :, :, 5] = q[0, :, :, 5].abs() + 0.1
    q[0, 0, 0, 9], q[0, 1, 1, 9] = 0.0, -1.0
    q[0, 2:, :, 9] = 1.0
    q[0, 0, 1, 9] = q[0, 1, 0, 9] = 1.0
    args[0][0, 0, 7, 5] = args[0][0, 0, 70, 9] = args[0][0, 0, 90, 5] = -math.inf
    mask = torch.eye(rows, dtype=torch.bool, device="cuda")
    mask[:, 0] = True
    got = ops.tree_attention(q, args[0], args[1], torch.tensor([90], device="cuda"), mask, scale=0.125)[0]
    spoilt = torch.zeros(rows, 2, dtype=torch.bool, device="cuda")
    spoilt[0, 0] = spoilt[1, 1] = True                       # 0 times, and -1 times, minus infinity
    want, bound = attended_by_row(q[0], args[0][0].double(), v[0], 90, mask, 0.125)
    assert bool(got[spoilt].isnan().all()) and bool(((got.double() - want).abs() <= bound)[~spoilt].all())
