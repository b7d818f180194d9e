"""Performance cases of the operators of speculative decoding: a drafted tree's rows are rotated, written into an
8-bit cache, attended to and verified.

Four kinds of pass, each through `dyninfer_b200.ops` where `own` is true and in elementary torch operations where it is not:

* `rotary` - rotary positions of a block of rows (query and key heads together, as a fused projection leaves them);
* `cache`  - new keys and values quantised into the rows of an 8-bit cache and the same rows read back as values;
* `attend` - a tree of drafted tokens (one token is the plain decode step) against the cached keys and values;
* `verify` - the drafted tree checked against the target's probabilities with given random numbers.

Head counts are those of the Qwen3 shapes of `dyninfer_b200.synth`, the vocabulary as well.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "q8": 1, "e4m3": 1}
CODES = {"q8": torch.int8, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # one step of a drafted chain on a small model: latency counts
        {"name": "rotary 5 rows", "kind": "rotary", "rows": 5, "heads": 24, "d": 128, "rot": 128, "layout": "half", "type": "f32",
         "scaling": "none", "factor": 1.0, "first": 600},
        # a prompt's chunk of a larger model
        {"name": "rotary 2048 rows", "kind": "rotary", "rows": 2048, "heads": 40, "d": 128, "rot": 128, "layout": "half",
         "type": "bf16", "scaling": "none", "factor": 1.0, "first": 0},
        # a document far into a lengthened context, half of the head in the interleaved layout
        {"name": "rotary 5003 rows far", "kind": "rotary", "rows": 5003, "heads": 72, "d": 128, "rot": 64,
         "layout": "interleaved", "type": "f32", "scaling": "yarn", "factor": 8.0, "first": 200000},
        # the new rows of 64 sequences' decode step
        {"name": "cache q8 64 x 1", "kind": "cache", "slots": 64, "rows": 1, "kv": 8, "d": 128, "cap": 2048, "type": "f32", "cache": "q8"},
        # eight prompts
        {"name": "cache e4m3 8 x 2048", "kind": "cache", "slots": 8, "rows": 2048, "kv": 8, "d": 128, "cap": 2304, "type": "bf16",
         "cache": "e4m3"},
        # a drafted chain in a chat, the framework's usual cache type
        {"name": "attend 1 x 5 at 600", "kind": "attend", "slots": 1, "rows": 5, "heads": 16, "kv": 8, "d": 128, "len": 600,
         "type": "f32", "cache": "bf16", "tree": False},
        # a few users with small trees
        {"name": "attend 8 x 13 at 2048", "kind": "attend", "slots": 8, "rows": 13, "heads": 32, "kv": 8, "d": 128, "len": 2048,
         "type": "f32", "cache": "q8", "tree": True},
        # large trees over long contexts
        {"name": "attend 4 x 64 at 8192", "kind": "attend", "slots": 4, "rows": 64, "heads": 32, "kv": 8, "d": 128, "len": 8192,
         "type": "bf16", "cache": "e4m3", "tree": True},
        # single tokens over very long contexts
        {"name": "attend 8 x 1 at 32768", "kind": "attend", "slots": 8, "rows": 1, "heads": 64, "kv": 8, "d": 128, "len": 32768,
         "type": "f16", "cache": "q8", "tree": False},
        # one user's chain, drafted by a smaller model
        {"name": "verify 1 x 5", "kind": "verify", "slots": 1, "rows": 5, "vocab": 151936, "type": "f32", "draft": True, "tree": False},
        # many users' trees without the draft's probabilities
        {"name": "verify 64 x 21 tree", "kind": "verify", "slots": 64, "rows": 21, "vocab": 151936, "type": "bf16", "draft": False,
         "tree": True},
        # trees drawn from a smaller model's probabilities
        {"name": "verify 32 x 13 tree drawn", "kind": "verify", "slots": 32, "rows": 13, "vocab": 151936, "type": "f32", "draft": True,
         "tree": True},
    ]


def _log(rng, low, high):
    """A whole number between the two, spread evenly over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["rotary", "cache", "attend", "attend", "verify"])
    if kind == "rotary":
        d = rng.choice([64, 80, 96, 128])
        heads = rng.choice([8, 10, 24, 40, 72])
        rot = rng.choice([d, d, d // 2, 2 * rng.randrange(1, d // 2 + 1)])
        scaling = rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]) if rot > 2 else "none"
        return {"kind": kind, "rows": _log(rng, 1, 5003 * 72 * 128 // (heads * d)), "heads": heads, "d": d, "rot": rot,
                "layout": rng.choice(["half", "interleaved"]), "type": rng.choice(["f32", "bf16", "f16"]), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]), "first": _log(rng, 1, 500000)}
    if kind == "cache":
        slots, kv, d = _log(rng, 1, 64), rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 96, 128])
        rows = _log(rng, 1, max(1, min(4096, (8 * 2048 * 8 * 128) // (slots * kv * d))))
        kind_type = rng.choice(["f32", "bf16", "f16"])
        rows = max(1, rows // 2) if kind_type == "f32" else rows
        return {"kind": kind, "slots": slots, "rows": rows, "kv": kv, "d": d, "cap": rows + rng.randrange(1, 300), "type": kind_type,
                "cache": rng.choice(["q8", "e4m3"])}
    if kind == "attend":
        cache, d = rng.choice(["bf16", "f16", "q8", "q8", "e4m3"]), rng.choice([64, 80, 96, 128, 128])
        kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        slots, rows = _log(rng, 1, 32), _log(rng, 1, 64)
        most = min(32768, 500_000_000 // (2 * slots * kv * d * SIZE[cache]), 8_600_000_000 // (slots * rows * kv * group * d))
        return {"kind": kind, "slots": slots, "rows": rows, "heads": kv * group, "kv": kv, "d": d, "len": _log(rng, 1, max(2, most)),
                "type": rng.choice(["f32", "bf16", "f16"]), "cache": cache, "tree": rng.random() < 0.7}
    draft, vocab = rng.random() < 0.5, _log(rng, 1000, 151936)
    slots = _log(rng, 1, 64)
    rows = _log(rng, 1, max(1, min(32, 32 * 13 * 151936 // (slots * vocab))))
    return {"kind": kind, "slots": slots, "rows": rows, "vocab": vocab, "type": rng.choice(["f32", "bf16", "f16"]), "draft": draft,
            "tree": rng.random() < 0.7}


class _State:
    pass


def _tree(case, rng):
    """Parents [slots, rows] of drafted trees: node 0 is the last token of the text, a node stands behind its parent."""
    slots, rows = case["slots"], case["rows"]
    parents = np.arange(rows)[None].repeat(slots, 0) - 1
    if case["tree"]:
        # a node goes under one of the last few before it: branches of several levels
        back = rng.integers(1, 5, size=(slots, rows))
        parents[:, 1:] = np.maximum(0, np.arange(1, rows) - back[:, 1:])
    return parents


def _ancestors(parents):
    """mask[slot, i, j]: node j is i or an ancestor of i."""
    slots, rows = parents.shape
    mask = np.zeros((slots, rows, rows), bool)
    for i in range(rows):
        at = parents[:, i]
        mask[:, i] = np.where((at >= 0)[:, None], mask[np.arange(slots), np.maximum(at, 0)], False)
        mask[:, i, i] = True
    return mask


def prepare(case, seed):
    s = _State()
    s.case = case
    gen = torch.Generator("cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    kind = case["kind"]
    if kind == "rotary":
        # query and key heads are the first ones of the fused projection's [q | k | v] rows
        total = case["heads"] + max(1, case["heads"] // 5)
        s.x = normal(case["rows"], total, case["d"]).to(TYPES[case["type"]])[:, :case["heads"]]
        # consecutive rows, now and then two at the same depth of a tree
        steps = torch.from_numpy((rng.random(case["rows"]) < 0.9).astype(np.int64)).cuda()
        s.positions = case["first"] + steps.cumsum(0)
        s.frequencies, s.magnitude = _frequencies(case)
    elif kind == "cache":
        shape = (case["slots"], case["rows"], case["kv"], case["d"])
        # channels of keys differ in size
        channel = normal(case["kv"], case["d"]).abs() + 0.2
        s.k, s.v = (normal(*shape) * channel).to(TYPES[case["type"]]), normal(*shape).to(TYPES[case["type"]])
        s.starts = torch.from_numpy(rng.integers(0, case["cap"] - case["rows"] + 1, size=case["slots"])).cuda()
        whole = (case["slots"], case["kv"], case["cap"])
        s.k_codes, s.v_codes = (torch.zeros(*whole, case["d"], device="cuda", dtype=torch.int8).view(CODES[case["cache"]]) for _ in "kv")
        s.k_scale, s.v_scale = (torch.zeros(*whole, device="cuda") for _ in "kv")
    elif kind == "attend":
        slots, rows, length = case["slots"], case["rows"], case["len"]
        s.q = (1.5 * normal(slots, rows, case["heads"], case["d"])).to(TYPES[case["type"]])
        # sequences of different ages
        lengths = rng.integers(-(-length * 3 // 4), length + 1, size=slots)
        lengths[0] = length
        s.lengths = torch.from_numpy(lengths).cuda()
        s.mask = torch.from_numpy(_ancestors(_tree(case, rng))).cuda()
        shape = (slots, case["kv"], length + rows, case["d"])
        s.k_scale = s.v_scale = None
        if case["cache"] in CODES:
            s.k, s.v = torch.empty(shape, device="cuda", dtype=CODES[case["cache"]]), torch.empty(shape, device="cuda", dtype=CODES[case["cache"]])
            s.k_scale, s.v_scale = torch.empty(shape[:3], device="cuda"), torch.empty(shape[:3], device="cuda")
            for slot in range(slots):
                for codes, scale in ((s.k, s.k_scale), (s.v, s.v_scale)):
                    codes[slot], scale[slot] = _quantised(normal(*shape[1:]), case["cache"])
        else:
            s.k, s.v = normal(*shape).to(TYPES[case["cache"]]), normal(*shape).to(TYPES[case["cache"]])
    else:
        slots, rows, vocab = case["slots"], case["rows"], case["vocab"]
        parents = _tree(case, rng)
        target, draft = (torch.empty(slots, rows, vocab, device="cuda", dtype=TYPES[case["type"]]) for _ in "pq")
        tokens = torch.zeros(slots, rows, device="cuda", dtype=torch.int64)
        for slot in range(slots):
            logits = 3 * normal(rows, vocab)
            target[slot] = torch.softmax(logits, -1)
            q = torch.softmax(0.9 * logits + 0.7 * normal(rows, vocab), -1)
            draft[slot] = q
            up = torch.from_numpy(np.maximum(parents[slot], 0)).cuda()
            if case["draft"]:
                # every node's token is drawn from the draft behind its parent
                tokens[slot] = torch.multinomial(q[up], 1, generator=gen)[:, 0]
            else:
                # siblings are the draft's best tokens, one after the other
                rank = [int((parents[slot, :i] == parents[slot, i]).sum()) for i in range(rows)]
                tokens[slot] = q.topk(min(vocab, 8), -1).indices[up, torch.tensor(rank, device="cuda")]
        s.tokens, s.parents = tokens, torch.from_numpy(parents).cuda()
        s.target, s.draft = target, draft if case["draft"] else None
        s.uniforms = torch.rand(slots, rows, generator=gen, device="cuda")
    return s


def _frequencies(case):
    """Inverse frequencies [rot / 2] in 64 bits on the host, and the factor of yarn on the rotated values."""
    rot, theta, factor, original = case["rot"], 1e6, case["factor"], 32768
    i = torch.arange(rot // 2, dtype=torch.float64)
    if case["scaling"] == "ntk":
        theta = theta * factor ** (rot / (rot - 2))
    f = theta ** (-2 * i / rot)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":
        # dimensions of over 32 turns in the original context stay, those of under one are stretched
        low, high = (rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1
    if case["scaling"] == "wavelength":
        # smooth between four turns and one turn in the original context
        smooth = ((original * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return (1 - smooth) * f / factor + smooth * f, 1.0
    return f, 1.0


def _quantised(x, kind):
    """(codes, scales) of rows along the last dimension."""
    x = x.float()
    top = x.abs().amax(-1)
    if kind == "q8":
        scale = (top.double() / 127).float()
        inverse = (127 / top.double()).float()
        # the product in 64 bits: next to a half, 32 would round twice
        return torch.round(x.double() * inverse[..., None].double()).to(torch.int8), scale
    # the least power of two under which the largest value fits 448 = 1.75 * 2^8
    fraction, exponent = torch.frexp(top)
    scale = torch.ldexp(torch.ones_like(top), exponent - 9 + (fraction > 0.875))
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def run(state):
    case = state.case
    if case["kind"] == "rotary":
        if own:
            from dyninfer_b200 import ops
            return ops.rotary(state.x, state.positions, state.frequencies, layout=case["layout"], magnitude=state.magnitude)
        return _rotary(state, case)
    if case["kind"] == "cache":
        where = state.k_codes, state.v_codes, state.k_scale, state.v_scale
        if own:
            from dyninfer_b200 import ops
            ops.kv_write(state.k, state.v, state.starts, *where)
            return ops.kv_read(state.starts, case["rows"], *where, dtype=TYPES[case["type"]])
        return _cache(state, case, where)
    if case["kind"] == "attend":
        if own:
            from dyninfer_b200 import ops
            return ops.tree_attention(state.q, state.k, state.v, state.lengths, state.mask, state.k_scale, state.v_scale)
        return _attend(state, case)
    if own:
        from dyninfer_b200 import ops
        return ops.verify_draft(state.tokens, state.parents, state.target, state.uniforms, state.draft)
    return _verify(state, case)


def _rotary(state, case):
    rot, x = case["rot"], state.x.float()
    angle = state.positions.double()[:, None] * state.frequencies.cuda()     # far positions: 64 bits
    cos, sin = (state.magnitude * angle.cos()).float()[:, None], (state.magnitude * angle.sin()).float()[:, None]
    if case["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1).to(state.x.dtype)


def _cache(state, case, where):
    k_codes, v_codes, k_scale, v_scale = where
    slot = torch.arange(case["slots"], device="cuda")[:, None, None]
    head = torch.arange(case["kv"], device="cuda")
    at = slot, head, (state.starts[:, None] + torch.arange(case["rows"], device="cuda"))[..., None]
    for x, codes, scales in ((state.k, k_codes, k_scale), (state.v, v_codes, v_scale)):
        new, scale = _quantised(x, case["cache"])
        codes.view(torch.int8)[at] = new.view(torch.int8)
        scales[at] = scale
    return tuple((codes.view(torch.int8)[at].view(codes.dtype).float() * scales[at][..., None]).to(TYPES[case["type"]])
                 for codes, scales in ((k_codes, k_scale), (v_codes, v_scale)))


def _attend(state, case):
    slots, rows, kv, d = case["slots"], case["rows"], case["kv"], case["d"]
    k, v = state.k.float(), state.v.float()
    if state.k_scale is not None:
        k, v = k * state.k_scale[..., None], v * state.v_scale[..., None]
    keys = k.shape[2]
    # which of its own tree's nodes a row sees, at the places where the tree stands in the cache
    j = torch.arange(keys, device="cuda") - state.lengths[:, None]
    node = j.clamp(0, rows - 1)[:, None].expand(slots, rows, keys)
    seen = (j < 0)[:, None] | ((j >= 0) & (j < rows))[:, None] & state.mask.gather(2, node)
    q = state.q.float().view(slots, rows, kv, -1, d).permute(0, 2, 3, 1, 4)       # [slots, kv, group, rows, d]
    group = q.shape[2]
    scores = torch.matmul(q.reshape(slots, kv, group * rows, d), k.transpose(2, 3)) / math.sqrt(d)
    scores = scores.view(slots, kv, group, rows, keys).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(slots, kv, group * rows, keys), v).view(slots, kv, group, rows, d)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 3, 1, 2, 4).reshape(slots, rows, kv * group, d).to(state.q.dtype)


def _verify(state, case):
    slots, rows = case["slots"], case["rows"]
    each = torch.arange(slots, device="cuda")
    tokens, u = state.tokens, state.uniforms.double()
    node = torch.zeros(slots, dtype=torch.int64, device="cuda")
    weight = state.target[:, 0].double()            # sums over the vocabulary and what is next to a border: 64 bits
    total = torch.ones(slots, dtype=torch.float64, device="cuda")
    count = torch.zeros_like(node)
    nodes = torch.full((slots, rows), -1, dtype=torch.int64, device="cuda")
    nodes[:, 0] = 0
    for i in range(1, rows):
        token = tokens[:, i]
        tried = state.parents[:, i] == node
        has = weight[each, token]
        if state.draft is None:
            taken = tried & (u[:, i] * total < has)
            left = weight.clone()
            left[each, token] = 0
            rest = total - has
        else:
            drafted = state.draft[each, node].double()
            taken = tried & (u[:, i] * drafted[each, token] * total < has)
            left = torch.where(total[:, None] > 0, weight / total[:, None], 0.0).sub(drafted).clamp(min=0)
            rest = left.sum(-1)
        refused = tried & ~taken
        weight = torch.where(taken[:, None], state.target[:, i].double(), torch.where(refused[:, None], left, weight))
        total = torch.where(taken, 1.0, torch.where(refused, rest, total))
        node = torch.where(taken, i, node)
        count = count + taken
        nodes[each, count] = node
    weight = torch.where((weight.sum(-1) == 0)[:, None], state.target[each, node].double(), weight)
    sums = weight.cumsum(-1)
    border = u[:, :1] * sums[:, -1:]
    beyond = sums > border
    last = weight.shape[1] - 1 - (weight > 0).flip(1).to(torch.int8).argmax(1)
    token = torch.where(beyond.any(1), beyond.to(torch.int8).argmax(1), last)
    fine = torch.isfinite(sums[:, -1]) & (sums[:, -1] > 0)
    return count, nodes, torch.where(fine, token, -1)


def work(case):
    size = SIZE[case["type"]]
    if case["kind"] == "rotary":
        n = case["rows"] * case["heads"] * case["d"]
        return {"bytes": 2 * n * size + 8 * case["rows"], "flops": 3 * case["rows"] * case["heads"] * case["rot"]}
    if case["kind"] == "cache":
        n = 2 * case["slots"] * case["rows"] * case["kv"]      # rows of keys and values
        # values in, codes and scales out, codes and scales in, values out
        return {"bytes": n * (2 * case["d"] * size + 2 * (case["d"] + 4)) + 16 * case["slots"], "flops": 4 * n * case["d"]}
    if case["kind"] == "attend":
        keys = case["slots"] * (case["len"] * 7 / 8 + case["rows"])
        row = case["d"] * SIZE[case["cache"]] + (4 if case["cache"] in CODES else 0)
        n = case["slots"] * case["rows"] * case["heads"] * case["d"]
        return {"bytes": 2 * keys * case["kv"] * row + 2 * n * size + case["slots"] * case["rows"] ** 2,
                "flops": 4 * case["rows"] * case["heads"] * case["d"] * keys}
    # the row that the last token is drawn from, and the draft's where a token was refused; the tests' single entries are nothing beside it
    n = case["slots"] * case["vocab"] * (2 if case["draft"] else 1)
    return {"bytes": n * size + case["slots"] * case["rows"] * 32, "flops": 2 * n}


def exact(case, seed):
    """What run() returns, from the definitions, in 64 bits."""
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        half, out = case["rot"] // 2, s.x.double().clone()
        first = slice(0, half) if case["layout"] == "half" else slice(0, case["rot"], 2)
        second = slice(half, case["rot"]) if case["layout"] == "half" else slice(1, case["rot"], 2)
        number = torch.complex(out[..., first].contiguous(), out[..., second].contiguous())
        angle = torch.outer(s.positions.double(), s.frequencies.to("cuda"))
        number = number * torch.polar(torch.full_like(angle, s.magnitude), angle)[:, None]
        out[..., first], out[..., second] = number.real, number.imag
        return out
    if case["kind"] == "cache":
        read = []
        for x in (s.k.double(), s.v.double()):
            top = x.abs().max(-1, keepdim=True).values
            if case["cache"] == "q8":
                step, per = (top / 127).float().double(), (127 / top).float().double()
                read.append(torch.round(x * per) * step)
            else:
                step = torch.exp2(torch.ceil(torch.log2(top / 448)))
                step = torch.where(top > 448 * step, 2 * step, step)
                step = torch.where(top <= 224 * step, step / 2, step)
                y = x / step
                unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                read.append(torch.round(y / unit) * unit * step)
        return tuple(read)
    if case["kind"] == "attend":
        slots, rows, heads, kv, d = (case[n] for n in ("slots", "rows", "heads", "kv", "d"))
        out = torch.zeros(slots, rows, heads, d, dtype=torch.float64, device="cuda")
        for b in range(slots):
            n = int(s.lengths[b])
            seen = torch.cat([torch.ones(rows, n, dtype=torch.bool, device="cuda"), s.mask[b]], 1)
            for g in range(kv):
                keys, values = s.k[b, g, :n + rows].double(), s.v[b, g, :n + rows].double()
                if s.k_scale is not None:
                    keys, values = keys * s.k_scale[b, g, :n + rows, None].double(), values * s.v_scale[b, g, :n + rows, None].double()
                for h in range(g * heads // kv, (g + 1) * heads // kv):
                    scores = (s.q[b, :, h].double() @ keys.T / math.sqrt(d)).masked_fill(~seen, -math.inf)
                    out[b, :, h] = torch.softmax(scores, -1) @ values
        return out
    counts, paths, drawn = [], [], []
    parents, tokens, u = s.parents.tolist(), s.tokens.tolist(), s.uniforms.double().tolist()
    for b in range(case["slots"]):
        path, i = [0], 1
        left, norm = s.target[b, 0].double(), 1.0
        while i < case["rows"]:
            if parents[b][i] == path[-1]:
                x = tokens[b][i]
                q = None if s.draft is None else s.draft[b, path[-1]].double()
                if u[b][i] * norm * (1.0 if q is None else float(q[x])) < float(left[x]):
                    path.append(i)
                    left, norm = s.target[b, i].double(), 1.0
                elif q is None:
                    norm -= float(left[x])
                    left = left.index_fill(0, torch.tensor([x], device="cuda"), 0.0)
                else:
                    left = torch.relu(left / norm - q) if norm > 0 else torch.zeros_like(left)
                    norm = float(left.sum())
            i += 1
        if float(left.sum()) == 0:
            left = s.target[b, path[-1]].double()
        sums = torch.cumsum(left, 0)
        drawn.append(int(torch.searchsorted(sums, u[b][0] * sums[-1:], right=True)))
        counts.append(len(path) - 1)
        paths.append(path + [-1] * (case["rows"] - len(path)))
    return torch.tensor(counts, device="cuda"), torch.tensor(paths, device="cuda"), torch.tensor(drawn, device="cuda")
