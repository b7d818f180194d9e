"""Host side of the operators of speculative decoding: refusals, which answer before any device is touched, and frequencies."""
import ctypes as C
import math
import os
import re

import pytest
import torch

from dyninfer_b200 import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def refused(kind, text, call, *args, **kwargs):
    with pytest.raises(kind, match=text):
        call(*args, **kwargs)


X = torch.zeros(3, 2, 8)
P = torch.arange(3)
F = torch.ones(4, dtype=torch.float64)


def test_rotary_refusals(native_lib):
    refused(TypeError, "float32, float16 or bfloat16", ops.rotary, X.double(), P, F)
    refused(ValueError, "layout", ops.rotary, X, P, F, layout="pairs")
    refused(ValueError, r"\[rows, heads, d\]", ops.rotary, X[0], P, F)
    refused(ValueError, "float64", ops.rotary, X, P, F.float())
    refused(ValueError, "positions", ops.rotary, X, P[:2], F)
    refused(TypeError, "positions must be int64", ops.rotary, X, P.float(), F)
    refused(ValueError, "dense", ops.rotary, torch.zeros(3, 2, 16)[..., ::2], P, F)
    refused(ValueError, "out must", ops.rotary, X, P, F, out=torch.zeros(3, 2, 8, dtype=torch.float16))
    refused(ValueError, "CUDA device", ops.rotary, X, P, F)


def cache(d=16, dtype=torch.int8, slots=2, heads=2, cap=4):
    codes = [torch.zeros(slots, heads, cap, d, dtype=torch.int8).view(dtype) for _ in "kv"]
    return (*codes, torch.zeros(slots, heads, cap), torch.zeros(slots, heads, cap))


def test_cache_refusals(native_lib):
    k = torch.zeros(2, 3, 2, 16)
    starts = torch.zeros(2, dtype=torch.int64)
    whole = cache()
    refused(TypeError, "k and v must both", ops.kv_write, k, k.half(), starts, *whole)
    refused(TypeError, "int8 or float8", ops.kv_write, k, k, starts, whole[0].float(), whole[1].float(), *whole[2:])
    refused(ValueError, "v has shape", ops.kv_write, k, k[:, :2], starts, *whole)
    refused(ValueError, "k has shape", ops.kv_write, k[:1], k[:1], starts, *whole)
    refused(ValueError, "starts", ops.kv_write, k, k, starts[:1], *whole)
    refused(ValueError, "counts", ops.kv_write, k, k, starts, *whole, counts=starts[:1])
    refused(ValueError, "k_scale", ops.kv_write, k, k, starts, whole[0], whole[1], whole[2][:, :1], whole[3])
    refused(TypeError, "v_scale must be float32", ops.kv_write, k, k, starts, *whole[:3], whole[3].half())
    refused(ValueError, "CUDA device", ops.kv_write, k, k, starts, *whole)
    refused(TypeError, "dtype", ops.kv_read, starts, 3, *whole, dtype=torch.float64)
    refused(ValueError, "at least zero", ops.kv_read, starts, -1, *whole)
    refused(ValueError, "CUDA device", ops.kv_read, starts, 3, *whole)


def test_tree_attention_refusals(native_lib):
    q, lengths = torch.zeros(2, 3, 4, 16), torch.zeros(2, dtype=torch.int64)
    whole = cache()
    plain = torch.zeros(2, 2, 4, 16, dtype=torch.bfloat16)
    refused(TypeError, "q must be", ops.tree_attention, q.double(), plain, plain, lengths)
    refused(TypeError, "caches must both", ops.tree_attention, q, plain.float(), plain.float(), lengths)
    refused(TypeError, "k_scale must be float32", ops.tree_attention, q, whole[0], whole[1], lengths)
    refused(ValueError, "no scales", ops.tree_attention, q, plain, plain, lengths, None, *whole[2:])
    refused(ValueError, "q has shape", ops.tree_attention, q[:1], plain, plain, lengths)
    refused(ValueError, "v_cache", ops.tree_attention, q, plain, plain[:1], lengths)
    refused(TypeError, "mask must be bool", ops.tree_attention, q, plain, plain, lengths, torch.zeros(3, 3))
    refused(ValueError, "mask has shape", ops.tree_attention, q, plain, plain, lengths, torch.zeros(4, 3, dtype=torch.bool))
    refused(ValueError, "dense", ops.tree_attention, q, plain.transpose(2, 3), plain.transpose(2, 3), lengths)
    refused(ValueError, "CUDA device", ops.tree_attention, q, plain, plain, lengths)


def test_verify_refusals(native_lib):
    t, u = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    p = torch.full((2, 3, 7), 1 / 7)
    refused(ValueError, "target must be", ops.verify_draft, t, t, p[0], u)
    refused(TypeError, "target must be", ops.verify_draft, t, t, p.double(), u)
    refused(ValueError, "tokens", ops.verify_draft, t[:, :2], t, p, u)
    refused(ValueError, "parents", ops.verify_draft, t, t[:, 0], p, u)
    refused(TypeError, "tokens must be int64", ops.verify_draft, u, t, p, u)
    refused(TypeError, "uniforms must be float32", ops.verify_draft, t, t, p, u.double())
    refused(TypeError, "draft must have", ops.verify_draft, t, t, p, u, p.half())
    refused(ValueError, "draft has shape", ops.verify_draft, t, t, p, u, p[:, :2])
    refused(ValueError, "CUDA device", ops.verify_draft, t, t, p, u)


# ---- the C entries, with pointers that are never followed -------------------------------------------------------------
S3, S6, S4, S2 = ((C.c_int64 * n)(*[16] * n) for n in (3, 6, 4, 2))
AT = 4096       # an aligned address


def native_refusal(name, text, *args):
    assert getattr(_lib.lib(), "dyninfer_cuda_" + name)(*args) != 0
    assert text in _lib.last_error(), _lib.last_error()


def test_native_rotary_refusals(native_lib):
    f = (C.c_double * 4)(1.0, 1.0, 1.0, 1.0)
    at = C.addressof(f)
    native_refusal("rotary", "type 7", AT, 7, S3, AT, at, 8, 0, 1.0, 1, 1, 1, 8, AT, S3, None)
    native_refusal("rotary", "even number", AT, 0, S3, AT, at, 7, 0, 1.0, 1, 1, 1, 8, AT, S3, None)
    native_refusal("rotary", "even number", AT, 0, S3, AT, at, 8, 0, 1.0, 1, 1, 1, 6, AT, S3, None)
    native_refusal("rotary", "even number", AT, 0, S3, AT, at, 8, 0, 1.0, 1, 1, 1, 258, AT, S3, None)
    native_refusal("rotary", "bad shape", AT, 0, S3, AT, at, 8, 0, 1.0, -1, 1, 1, 8, AT, S3, None)
    native_refusal("rotary", "magnitude", AT, 0, S3, AT, at, 8, 0, math.inf, 1, 1, 1, 8, AT, S3, None)
    native_refusal("rotary", "NULL", None, 0, S3, AT, at, 8, 0, 1.0, 1, 1, 1, 8, AT, S3, None)
    native_refusal("rotary", "aligned", AT + 2, 0, S3, AT, at, 8, 0, 1.0, 1, 1, 1, 8, AT, S3, None)
    flat = (C.c_int64 * 3)(16, 0, 16)
    native_refusal("rotary", "stride 0", AT, 0, flat, AT, at, 8, 0, 1.0, 1, 2, 2, 8, AT, flat, None)
    f[2] = math.nan
    native_refusal("rotary", "frequency 2", AT, 0, S3, AT, at, 8, 0, 1.0, 1, 1, 1, 8, AT, S3, None)
    assert native_lib.dyninfer_cuda_rotary(None, 0, None, None, at, 8, 0, 1.0, 0, 1, 1, 8, None, None, None) == 0   # nothing to do


def test_native_cache_refusals(native_lib):
    def write(*, x=AT, type=0, codes=AT, kind=32, strides=S6, scale=AT, starts=AT, batch=1, rows=1, heads=1, d=16, cap=1):
        return (x, AT, type, S6, codes, AT, kind, strides, scale, AT, S4, starts, None, batch, rows, heads, d, cap, None)
    native_refusal("kv_write", "type 9", *write(type=9))
    native_refusal("kv_write", "not an 8-bit", *write(kind=1))
    native_refusal("kv_write", "head dim 24", *write(d=24))
    native_refusal("kv_write", "head dim 272", *write(d=272))
    native_refusal("kv_write", "bad shape", *write(cap=0))
    native_refusal("kv_write", "NULL", *write(scale=None))
    native_refusal("kv_write", "aligned", *write(x=AT + 2))
    native_refusal("kv_write", "multiples of 16", *write(codes=AT + 8))
    native_refusal("kv_write", "multiples of 16", *write(strides=(C.c_int64 * 6)(16, 16, 16, 16, 16, 24), cap=2))
    native_refusal("kv_write", "stride 0", *write(strides=(C.c_int64 * 6)(0, 16, 16, 0, 16, 16), batch=2))
    assert native_lib.dyninfer_cuda_kv_write(*write(x=None, rows=0)) == 0
    read = (AT, AT, 0, S6, AT, AT, 32, S6, AT, AT, S4, AT, 1, 1, 1, 24, 1, None)
    native_refusal("kv_read", "kv_read: head dim 24", *read)


def test_native_tree_attention_refusals(native_lib):
    def call(*, q=AT, type=0, k=AT, kind=32, strides=S6, ks=AT, lengths=AT, mask=None, ms=None, batch=1, rows=1, heads=2, kv=1, d=16,
             cap=4, scale=1.0, out=AT):
        return (q, type, S3, k, AT, kind, strides, ks, AT, S4, lengths, mask, ms, batch, rows, heads, kv, d, cap, scale, out, None)
    native_refusal("tree_attention", "query type", *call(type=5))
    native_refusal("tree_attention", "cache type 0", *call(kind=0))
    native_refusal("tree_attention", "head dim 136", *call(d=136))
    native_refusal("tree_attention", "multiple of kv heads", *call(heads=3, kv=2))
    native_refusal("tree_attention", "bad shape", *call(cap=0))
    for scale in (math.nan, math.inf, 0.0, -1.0):
        native_refusal("tree_attention", "scale must be above zero", *call(scale=scale))
    native_refusal("tree_attention", "needs its scales", *call(ks=None))
    native_refusal("tree_attention", "needs its strides", *call(mask=AT))
    native_refusal("tree_attention", "multiples of 16", *call(k=AT + 4))
    native_refusal("tree_attention", "multiples of 16", *call(kind=1, strides=(C.c_int64 * 6)(16, 16, 16, 16, 16, 12)))
    native_refusal("tree_attention", "NULL", *call(lengths=None))
    assert native_lib.dyninfer_cuda_tree_attention(*call(q=None, rows=0)) == 0


def test_native_verify_refusals(native_lib):
    def call(*, tokens=AT, target=AT, draft=None, ds=None, type=0, batch=1, nodes=2, vocab=7):
        return (tokens, AT, 0, target, S2, draft, ds, type, AT, batch, nodes, vocab, AT, AT, AT, None)
    native_refusal("verify_draft", "type 3", *call(type=3))
    native_refusal("verify_draft", "1 to 1024 nodes", *call(nodes=1025))
    native_refusal("verify_draft", "1 to 1024 nodes", *call(nodes=0))
    native_refusal("verify_draft", "bad shape", *call(vocab=0))
    native_refusal("verify_draft", "need their strides", *call(draft=AT))
    native_refusal("verify_draft", "NULL", *call(tokens=None))
    native_refusal("verify_draft", "aligned", *call(target=AT + 2))
    assert native_lib.dyninfer_cuda_verify_draft(*call(tokens=None, batch=0)) == 0


# ---- frequencies ------------------------------------------------------------------------------------------------------
def test_frequencies_and_their_scalings():
    rot, theta = 64, 1e6
    plain = [theta ** (-2 * i / rot) for i in range(rot // 2)]

    def near(got, want):
        assert got.dtype == torch.float64 and torch.allclose(got, torch.tensor(want, dtype=torch.float64), rtol=1e-13, atol=0)

    f, m = ops.rotary_frequencies(rot, theta)
    near(f, plain)
    assert m == 1.0
    near(ops.rotary_frequencies(rot, theta, "linear", 4.0)[0], [x / 4 for x in plain])
    f = ops.rotary_frequencies(rot, theta, "ntk", 4.0)[0]
    assert f[0] == 1.0 and abs(float(f[-1]) * 4 / plain[-1] - 1) < 1e-12      # the slowest is stretched by the factor
    f, m = ops.rotary_frequencies(rot, theta, "yarn", 4.0, original_length=32768)
    turns = [32768 * x / (2 * math.pi) for x in plain]
    assert abs(m - (0.1 * math.log(4) + 1)) < 1e-15
    for i, n in enumerate(turns):
        if n > 64:
            assert float(f[i]) == pytest.approx(plain[i], rel=1e-13)
        elif n < 0.5:
            assert float(f[i]) == pytest.approx(plain[i] / 4, rel=1e-13)
        assert plain[i] / 4 * (1 - 1e-13) <= float(f[i]) <= plain[i] * (1 + 1e-13)
    f, m = ops.rotary_frequencies(rot, theta, "wavelength", 8.0, original_length=8192)
    turns = [8192 * x / (2 * math.pi) for x in plain]
    keep = [min(1.0, max(0.0, (n - 1) / 3)) for n in turns]
    near(f, [x * k + x / 8 * (1 - k) for x, k in zip(plain, keep)])
    assert m == 1.0


@pytest.mark.parametrize("args,text", [((7,), "even"), ((0,), "even"), ((8, -1.0), "theta"), ((8, 1e4, "none", 0.0), "factor"),
                                       ((2, 1e4, "ntk", 2.0), "more than one pair"), ((8, 1e4, "cubic", 2.0), "not one of"),
                                       ((8, 1e4, "yarn", 2.0), "original_length"),
                                       ((8, 1e4, "yarn", 2.0, 4096, 5.0, 2.0), "below high")])
def test_frequency_refusals(args, text):
    refused(ValueError, text, ops.rotary_frequencies, *args)


def test_waits_that_run_out_are_reported_under_their_own_name():
    """Each file's bounded waits leave its own code in the device's error word, and the message names every code."""
    csrc = os.path.join(ROOT, "dyninfer_b200", "csrc")
    text = {f: open(os.path.join(csrc, f)).read() for f in os.listdir(csrc)}
    codes = dict(re.findall(r"(DEV_ERR_\w+) = (\d+)", text["common.cuh"]))
    message = re.search(r"a bounded wait inside a kernel expired.*?\)", re.sub(r'"\s*"', "", text["api.cu"]))[0]
    assert len(codes) >= 3 and all(re.search(rf"\b{c} \w", message) for c in codes.values())
    for name, source in text.items():
        kind = "ATTENTION_PIPE" if name.startswith("attention") else "GEM"
        assert all(kind in c for c in re.findall(r"report_wait_expired\([^,()]+, (DEV_ERR_\w+)\)", source)), name
