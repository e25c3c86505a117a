"""Measured cases of the cached-decoding operators, with their plain forms.

The operators are the ones a decoder runs around its attention when it answers token by token, or
verifies a tree of drafted tokens: `rotary_embedding`, `qk_norm_rotary`, `qk_norm_rotary_append`,
`tree_attention` and `kv_cache_commit`.  `run` computes them in elementary torch operations, or, where
`own` is true, through `hackathon_b200.kernel_registry`.

Shapes: activations [batch, tokens, heads, head_dim]; caches [batch, kv_heads, capacity, head_dim];
`lengths[b]` rows of sequence b's cache are committed, the drafted tokens' rows follow them.
Rotary frequencies are phase steps: the fraction of a turn that one position adds, times 2**64.
"""

import math

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "f32": 4}
_EPS = 1e-6


# ------------------------------------------------------------------ cases

def _rotary(name, **k):
    return dict({"name": name, "op": "rotary", "interleaved": False, "base": 10000.0, "factor": 1.0}, **k)


def _norm(name, **k):
    return dict({"name": name, "op": "norm", "interleaved": False, "base": 10000.0, "factor": 1.0}, **k)


def _append(name, **k):
    return dict({"name": name, "op": "append", "interleaved": False, "base": 10000.0, "factor": 1.0}, **k)


def listed():
    return [
        # one new token of a small batch: a launch and little else
        _rotary("rotary_token", dtype="bf16", batch=8, tokens=1, heads=16, dim=64, rotary=64, start=900),
        # a long prompt's chunk far into a context stretched 32 times, half of each head rotated
        _rotary("rotary_far_chunk", dtype="fp16", batch=2, tokens=8191, heads=32, dim=128, rotary=64, start=500000,
                interleaved=True, base=500000.0, factor=32.0),
        # the prompt pass: the packed projection normalised and rotated ahead of the flash attention
        _norm("norm_prompt", dtype="bf16", batch=64, tokens=512, heads=32, kv_heads=8, dim=128, rotary=128, start=0),
        # the fp32 profile's prompt pass at the small decoder's head size
        _norm("norm_prompt_f32", dtype="f32", batch=16, tokens=128, heads=4, kv_heads=4, dim=64, rotary=64, start=0),
        # one token for each of a batch of sequences of different lengths, straight into the caches
        _append("append_token", dtype="bf16", batch=32, tokens=1, heads=32, kv_heads=8, dim=128, rotary=128,
                shortest=37, longest=1901),
        # drafted trees into the caches
        _append("append_tree", dtype="fp16", batch=24, tokens=63, heads=16, kv_heads=16, dim=64, rotary=64,
                shortest=0, longest=1023, interleaved=True),
        # one token, one short sequence: the smallest attention call
        {"name": "attend_token", "op": "tree", "dtype": "bf16", "batch": 1, "tokens": 1, "heads": 16, "kv_heads": 16,
         "dim": 64, "shortest": 130, "longest": 130},
        # the decode step of a batch of conversations
        {"name": "attend_batch", "op": "tree", "dtype": "bf16", "batch": 32, "tokens": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "shortest": 511, "longest": 7000},
        # one sequence with a very long context and a short chain of drafts
        {"name": "attend_long", "op": "tree", "dtype": "fp16", "batch": 1, "tokens": 5, "heads": 32, "kv_heads": 8,
         "dim": 128, "shortest": 131001, "longest": 131001},
        # wide trees over a batch: 512 query rows for each key and value head
        {"name": "attend_wide_tree", "op": "tree", "dtype": "bf16", "batch": 16, "tokens": 64, "heads": 64, "kv_heads": 8,
         "dim": 128, "shortest": 2000, "longest": 4100},
        # the fp32 profile's decode step
        {"name": "attend_f32", "op": "tree", "dtype": "f32", "batch": 8, "tokens": 3, "heads": 16, "kv_heads": 16,
         "dim": 64, "shortest": 0, "longest": 1000},
        # the accepted paths of a batch of trees move together
        {"name": "commit_batch", "op": "commit", "dtype": "bf16", "batch": 32, "tokens": 64, "kv_heads": 8, "dim": 128,
         "shortest": 0, "longest": 511, "path": 9},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "append", "tree", "tree", "tree", "commit"])
    c = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "f32"])}
    if op in ("rotary", "norm", "append"):
        c["dim"] = rng.choice([64, 64, 80, 96, 128, 128, 256])
        c["rotary"] = rng.choice([c["dim"], c["dim"], c["dim"] // 2, c["dim"] // 4])
        c["interleaved"] = rng.random() < 0.5
        c["base"], c["factor"] = rng.choice([(10000.0, 1.0), (500000.0, 1.0), (10000.0, 4.0), (500000.0, 32.0)])
        most = 48_000_000 // c["dim"]  # rows of head_dim values
        if op == "rotary":
            c["heads"] = rng.choice([1, 4, 8, 12, 16, 32])
        else:
            c["kv_heads"] = rng.choice([1, 2, 4, 8, 16])
            c["heads"] = c["kv_heads"] * rng.choice([1, 1, 3, 4, 8])
        width = c["heads"] + 2 * c.get("kv_heads", 0)
        c["tokens"] = _log(rng, 1, 128 if op == "append" else 8192)
        c["batch"] = _log(rng, 1, max(1, min(64, most // (width * c["tokens"]))))
        if op == "append":
            c["longest"] = _log(rng, 1, 1024 if c["dtype"] == "f32" else 2048)
            c["shortest"] = rng.randint(0, c["longest"])
        else:
            c["start"] = rng.choice([0, rng.randint(1, 4096), rng.randint(1, 1 << 20)])
        return c
    c["dim"] = rng.choice([64, 128])
    c["kv_heads"] = rng.choice([1, 2, 4, 8, 16])
    if op == "commit":
        c["batch"], c["tokens"] = _log(rng, 1, 64), _log(rng, 2, 128)
        c["path"] = rng.randint(1, min(16, c["tokens"]))
        c["longest"] = _log(rng, 1, 1024)
        c["shortest"] = rng.randint(0, c["longest"])
        return c
    c["heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 7, 8])
    c["tokens"] = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 64)])
    c["longest"] = _log(rng, 1, 100_000)
    rows = 300_000 if c["dtype"] != "f32" else 100_000  # cached rows of every kv head, 128 values each
    c["batch"] = _log(rng, 1, max(1, min(64, rows * 128 // (c["dim"] * c["kv_heads"] * c["longest"]))))
    c["shortest"] = rng.randint(0, c["longest"])
    return c


# ------------------------------------------------------------------ inputs

def _capacity(case):
    return case["longest"] + case["tokens"] + 3


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly apart."""
    return [lo + (hi - lo) * i // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _frequencies(case):
    """Radians a position, [rotary / 2], and the factor on sines and cosines: below a wavelength of
    4096 / 32 positions as trained, above 4096 slowed by `factor`, a linear ramp between (in turns)."""
    half = case["rotary"] // 2
    f = case["base"] ** (-np.arange(half, dtype=np.float64) / half)
    if case["factor"] == 1.0:
        return f, 1.0
    turns = 4096.0 * f / (2.0 * math.pi)
    keep = np.clip((turns - 1.0) / 31.0, 0.0, 1.0)
    return f * keep + f / case["factor"] * (1.0 - keep), 0.1 * math.log(case["factor"]) + 1.0


def _phase_steps(freq):
    """Turns a position times 2**64, as int64."""
    return torch.tensor([int(math.ldexp(float(v) / (2.0 * math.pi), 64)) for v in freq], dtype=torch.int64)


def _tree(rs, batch, tokens):
    """Random trees, parents before children: depth [batch, tokens] and who sees whom (itself and its
    ancestors) [batch, tokens, tokens]."""
    sees = np.zeros((batch, tokens, tokens), bool)
    depth = np.zeros((batch, tokens), np.int64)
    rows = np.arange(batch)
    for i in range(1, tokens):
        parent = rs.randint(max(0, i - 8), i, batch)
        sees[:, i] = sees[rows, parent]
        sees[rows, i, parent] = True
        depth[:, i] = depth[rows, parent] + 1
    sees[:, np.arange(tokens), np.arange(tokens)] = True
    return depth, sees


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 31))
    dt = _TYPES[case["dtype"]]

    def values(*shape):
        # written piece by piece into its own type, so no 32-bit copy of a whole cache is held
        out = torch.empty(shape, dtype=dt, device=dev)
        for piece in out.view(-1).split(1 << 27):
            piece.copy_(torch.randn(piece.shape, generator=gen, device=dev))
        return out

    s = {"case": dict(case)}
    b, t, d = case["batch"], case["tokens"], case["dim"]
    if case["op"] in ("rotary", "norm", "append"):
        freq, s["scale"] = _frequencies(case)
        s["steps"] = _phase_steps(freq).to(dev)
    if "longest" in case:
        lengths = rs.permutation(_spread(case["shortest"], case["longest"], b))
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
    if case["op"] == "rotary":
        s["x"] = values(b, t, case["heads"], d)
        s["out"] = torch.zeros_like(s["x"])
    elif case["op"] in ("norm", "append"):
        s["qkv"] = values(b, t, case["heads"] + 2 * case["kv_heads"], d)
        s["q_weight"] = 1.0 + 0.1 * torch.randn(d, generator=gen, device=dev)
        s["k_weight"] = 1.0 + 0.1 * torch.randn(d, generator=gen, device=dev)
    if "start" in case:
        first = case["start"] + rs.randint(0, 32, (b, 1))
        s["positions"] = torch.tensor(first + np.arange(t), dtype=torch.int64, device=dev)
    if case["op"] == "norm":
        s["out"] = torch.zeros_like(s["qkv"])
    if case["op"] in ("append", "tree", "commit"):
        shape = (b, case["kv_heads"], _capacity(case), d)
        s["k_cache"], s["v_cache"] = values(*shape), values(*shape)
    if case["op"] in ("append", "tree"):
        depth, sees = _tree(rs, b, t)
    if case["op"] == "append":
        s["positions"] = torch.tensor(lengths[:, None] + depth, dtype=torch.int64, device=dev)
        s["out"] = torch.zeros(b, t, case["heads"], d, dtype=dt, device=dev)
    elif case["op"] == "tree":
        s["q"] = values(b, t, case["heads"], d)
        s["tree_mask"] = torch.tensor(sees, device=dev)
        s["out"] = torch.zeros_like(s["q"])
    elif case["op"] == "commit":
        path = np.sort(np.argsort(rs.rand(b, t), axis=1)[:, : case["path"]], axis=1)
        s["path"] = torch.tensor(path, dtype=torch.int32, device=dev)
        s["accepted"] = torch.tensor(rs.permutation(_spread(0, case["path"], b)), dtype=torch.int32, device=dev)
        s["new_lengths"] = torch.zeros_like(s["lengths"])
    return s


# ------------------------------------------------------------------ plain forms

def _rotate(x, positions, steps, scale, interleaved):
    """x [batch, tokens, heads, dim] in 32 bits; the angles in 64."""
    turn = steps.double() * (2.0 * math.pi / 2.0 ** 64)
    angle = (positions.double().unsqueeze(-1) * turn).unsqueeze(2)
    cos, sin = (torch.cos(angle) * scale).float(), (torch.sin(angle) * scale).float()
    rot = 2 * steps.numel()
    head, tail = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = head[..., : rot // 2], head[..., rot // 2:]
        head = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((head, tail), -1)


def _normed(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight


def _plain_rotary(s):
    x = s["x"]
    return _rotate(x.float(), s["positions"], s["steps"], s["scale"], s["case"]["interleaved"]).to(x.dtype)


def _plain_split(s):
    qkv, c = s["qkv"], s["case"]
    q, k, v = qkv.split((c["heads"], c["kv_heads"], c["kv_heads"]), 2)
    more = (s["positions"], s["steps"], s["scale"], c["interleaved"])
    q = _rotate(_normed(q.float(), s["q_weight"]), *more).to(qkv.dtype)
    k = _rotate(_normed(k.float(), s["k_weight"]), *more).to(qkv.dtype)
    return q, k, v


def _plain_append(s):
    q, k, v = _plain_split(s)
    c = s["case"]
    b = torch.arange(c["batch"], device=q.device).unsqueeze(-1)
    at = s["lengths"].long().unsqueeze(-1) + torch.arange(c["tokens"], device=q.device)
    s["k_cache"][b, :, at] = k
    s["v_cache"][b, :, at] = v
    return q, s["k_cache"], s["v_cache"]


def _plain_tree(s):
    q, c = s["q"], s["case"]
    b, t, hk, d = c["batch"], c["tokens"], c["kv_heads"], c["dim"]
    g, n = c["heads"] // hk, s["k_cache"].shape[2]
    rows = q.float().view(b, t, hk, g, d).permute(0, 2, 1, 3, 4).reshape(b, hk, t * g, d)
    scores = rows @ s["k_cache"].float().transpose(-1, -2) / math.sqrt(d)
    draft = torch.arange(n, device=q.device) - s["lengths"].unsqueeze(-1)  # a cache row's place among the drafts
    among = ((draft >= 0) & (draft < t)).view(b, 1, n)
    sees = s["tree_mask"].gather(2, draft.clamp(0, t - 1).view(b, 1, n).expand(b, t, n))
    sees = (draft < 0).view(b, 1, n) | (among & sees)
    sees = sees.repeat_interleave(g, 1).unsqueeze(1)
    scores = torch.where(sees, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = p @ s["v_cache"].float() / torch.where(total == 0, 1.0, total)
    return out.view(b, hk, t, g, d).permute(0, 2, 1, 3, 4).reshape(b, t, hk * g, d).to(q.dtype)


def _plain_commit(s):
    a = s["path"].shape[1]
    b = torch.arange(s["path"].shape[0], device=s["path"].device).unsqueeze(-1)
    step = torch.arange(a, device=b.device)
    base = s["lengths"].long().unsqueeze(-1)
    source = base + torch.where(step < s["accepted"].unsqueeze(-1), s["path"].long(), step)  # behind the path: itself
    s["k_cache"][b, :, base + step] = s["k_cache"][b, :, source]
    s["v_cache"][b, :, base + step] = s["v_cache"][b, :, source]
    return s["k_cache"], s["v_cache"], s["lengths"] + s["accepted"]


_PLAIN = {"rotary": _plain_rotary, "norm": lambda s: torch.cat(_plain_split(s), 2), "append": _plain_append,
          "tree": _plain_tree, "commit": _plain_commit}


# ------------------------------------------------------------------ the framework's calls

def _own_rotary(s, kernel):
    outs = [s["out"]]
    kernel("rotary_embedding")([s["x"], s["positions"], s["steps"]], outs,
                               {"interleaved": int(s["case"]["interleaved"]), "scale": s["scale"]})
    return outs[0]


def _heads(s):
    c = s["case"]
    return {"num_heads": c["heads"], "kv_num_heads": c["kv_heads"], "epsilon": _EPS,
            "interleaved": int(c["interleaved"]), "scale": s["scale"]}


def _own_norm(s, kernel):
    outs = [s["out"]]
    kernel("qk_norm_rotary")([s["qkv"], s["q_weight"], s["k_weight"], s["positions"], s["steps"]], outs, _heads(s))
    return outs[0]


def _own_append(s, kernel):
    outs = [s["out"], s["k_cache"], s["v_cache"]]
    kernel("qk_norm_rotary_append")([s["qkv"], s["q_weight"], s["k_weight"], s["positions"], s["steps"], s["lengths"]],
                                    outs, _heads(s))
    return tuple(outs)


def _own_tree(s, kernel):
    outs = [s["out"]]
    kernel("tree_attention")([s["q"], s["k_cache"], s["v_cache"], s["lengths"], s["tree_mask"]], outs, {})
    return outs[0]


def _own_commit(s, kernel):
    outs = [s["k_cache"], s["v_cache"], s["new_lengths"]]
    kernel("kv_cache_commit")([s["lengths"], s["path"], s["accepted"]], outs, {})
    return tuple(outs)


_OWN = {"rotary": _own_rotary, "norm": _own_norm, "append": _own_append, "tree": _own_tree, "commit": _own_commit}


def run(state):
    if own:
        from hackathon_b200.kernel_registry import lookup
        return _OWN[state["case"]["op"]](state, lookup)
    return _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------ floors

def work(case):
    es, b, t, d = _BYTES[case["dtype"]], case["batch"], case["tokens"], case["dim"]
    if case["op"] == "rotary":
        n = b * t * case["heads"] * d
        return {"bytes": 2 * n * es + 8 * b * t, "flops": 3 * n}
    if case["op"] in ("norm", "append"):
        n = b * t * (case["heads"] + 2 * case["kv_heads"]) * d
        return {"bytes": 2 * n * es + 8 * b * t + 8 * d, "flops": 8 * n}
    if case["op"] == "commit":
        moved = sum(_spread(0, case["path"], b)) * case["kv_heads"] * d
        return {"bytes": 4 * moved * es + 4 * b * (case["path"] + 3), "flops": 0}
    rows = sum(n + t for n in _spread(case["shortest"], case["longest"], b))
    return {"bytes": 2 * rows * case["kv_heads"] * d * es + 2 * b * t * case["heads"] * d * es + b * t * t,
            "flops": 4 * rows * t * case["heads"] * d}


# ------------------------------------------------------------------ 64-bit definition

def _exact_turned(x, s):
    """x in 64 bits, each pair a complex number times scale * exp(i angle)."""
    half = s["steps"].numel()
    per = s["steps"].double() / 2.0 ** 64 * 2.0 * math.pi
    angle = (s["positions"].double()[:, :, None] * per[None, None])[:, :, None, :]
    w = torch.polar(torch.full_like(angle, s["scale"]), angle)
    out = x.clone()
    i = torch.arange(half, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if s["case"]["interleaved"] else (i, i + half)
    z = torch.complex(x[..., lo], x[..., hi]) * w
    out[..., lo], out[..., hi] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    b, t, d, hk = case["batch"], case["tokens"], case["dim"], case.get("kv_heads", 0)
    if case["op"] == "rotary":
        return _exact_turned(s["x"].double(), s)
    if case["op"] in ("norm", "append"):
        x = s["qkv"].double()
        h = case["heads"]
        unit = x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + _EPS)
        q = _exact_turned(unit[:, :, :h] * s["q_weight"].double(), s)
        k = _exact_turned(unit[:, :, h:h + hk] * s["k_weight"].double(), s)
        if case["op"] == "norm":
            return torch.cat((q, k, x[:, :, h + hk:]), 2)
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for i, n in enumerate(s["lengths"].tolist()):
            kc[i, :, n:n + t] = k[i].transpose(0, 1)
            vc[i, :, n:n + t] = x[i, :, h + hk:].transpose(0, 1)
        return q, kc, vc
    if case["op"] == "commit":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for i, (n, m) in enumerate(zip(s["lengths"].tolist(), s["accepted"].tolist())):
            rows = (n + s["path"][i, :m]).long()
            kc[i, :, n:n + m] = kc[i][:, rows]
            vc[i, :, n:n + m] = vc[i][:, rows]
        return kc, vc, None
    out = torch.zeros(b, t, hk, case["heads"] // hk, d, dtype=torch.float64, device=s["q"].device)
    for i, n in enumerate(s["lengths"].tolist()):
        hidden = torch.zeros(t, n + t, dtype=torch.bool, device=out.device)
        hidden[:, n:] = ~s["tree_mask"][i]
        for j in range(hk):
            q = s["q"][i].view(t, hk, -1, d)[:, j].double()
            k, v = s["k_cache"][i, j, :n + t].double(), s["v_cache"][i, j, :n + t].double()
            e = torch.einsum("tgd,nd->tgn", q, k) * d ** -0.5
            e.masked_fill_(hidden.unsqueeze(1), -math.inf)
            e = (e - e.amax(-1, keepdim=True)).exp()
            out[i, :, j] = torch.einsum("tgn,nd->tgd", e, v) / e.sum(-1, keepdim=True)
    return out.view(b, t, case["heads"], d)
