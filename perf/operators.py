"""Workloads of the few-token MoE layer and of the low-rank adapters beside a shared projection.

`listed()` names the cases, `draw()` makes more of the same ranges, `prepare()` builds what a program has in hand before the call and
`run()` makes one pass: through the package's entry points where `own` is true, else through the same operators spelled
out in elementary 32-bit tensor operations. `exact()` is the operators' definition in 64 bits.

kind "mlp"      few_token_mlp: the expert MLP of a layer, router outputs given (T tokens, k slots each)
kind "moe"      few_token_moe: the same layer with its router
kind "adapter"  adapter_linear, forward: shared projection plus the token's own low-rank adapter
kind "train"    adapter_linear, forward and backward: gradients of the input and of the adapters (and of the shared
                weight and bias where the case has them)
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# how the activation reads the up-projection: one column per hidden value, halves with the second or the first
# one activated, or interleaved gate / up columns with the clamped SwiGLU
LAYOUTS = {"plain": 0, "glu_second": 1, "glu_first": 2, "interleaved": 3}
ACTS = {"silu": 0, "gelu": 1}
ALPHA, LIMIT = 1.702, 7.0


def listed():
    return [
        # One decoding stream on a layer of many small experts: 8 experts of 4.7 MB, latency counts.
        {"name": "one token, 64 small experts", "kind": "mlp", "dtype": "bf16", "T": 1, "d": 1536, "F": 512, "E": 64, "k": 8,
         "layout": "glu_first", "act": "silu", "bias": False, "order": "out_in", "padded": 0},
        # One decoding stream on large experts: two of them, 352 MB each, a plain stream of weights.
        {"name": "one token, 8 large experts", "kind": "mlp", "dtype": "bf16", "T": 1, "d": 4096, "F": 14336, "E": 8, "k": 2,
         "layout": "glu_second", "act": "silu", "bias": False, "order": "out_in", "padded": 0},
        # A serving batch on the same layer: every expert is active with about 16 rows.
        {"name": "64 tokens, 8 large experts", "kind": "mlp", "dtype": "bf16", "T": 64, "d": 4096, "F": 14336, "E": 8, "k": 2,
         "layout": "glu_second", "act": "silu", "bias": False, "order": "out_in", "padded": 0},
        # A serving batch with the router, 128 experts of which most are active with one to four rows.
        {"name": "24 tokens, router, 128 experts", "kind": "moe", "dtype": "fp16", "T": 24, "d": 2048, "F": 768, "E": 128, "k": 8,
         "layout": "glu_first", "act": "silu", "bias": False, "order": "out_in", "mode": "softmax_topk"},
        # Weights stored input-major with biases everywhere and the clamped interleaved activation.
        {"name": "16 tokens, router, biases", "kind": "moe", "dtype": "bf16", "T": 16, "d": 2880, "F": 2880, "E": 32, "k": 4,
         "layout": "interleaved", "act": "silu", "bias": True, "order": "in_out", "mode": "topk_softmax"},
        # A small layer in 32 bits with sizes no vector width divides, in a batch padded by three empty rows.
        {"name": "11 tokens, odd sizes, 32 bits", "kind": "mlp", "dtype": "fp32", "T": 11, "d": 1001, "F": 427, "E": 13, "k": 3,
         "layout": "plain", "act": "gelu", "bias": True, "order": "out_in", "padded": 3},
        # One decoding stream through an adapted projection.
        {"name": "adapter, one token", "kind": "adapter", "dtype": "bf16", "T": 1, "in": 4096, "out": 4096, "r": 16, "n": 32,
         "bias": False, "order": "segments", "requests": 1, "bare": 0.0},
        # A decoding batch in which nearly every request brings its own adapter and some bring none.
        {"name": "adapter, 61 requests", "kind": "adapter", "dtype": "fp16", "T": 61, "in": 2048, "out": 4096, "r": 32, "n": 64,
         "bias": True, "order": "shuffled", "requests": 61, "bare": 0.1},
        # The prompts of six requests in one batch, lengths ragged.
        {"name": "adapter, prompts of 6 requests", "kind": "adapter", "dtype": "bf16", "T": 4099, "in": 4096, "out": 4096, "r": 16,
         "n": 16, "bias": False, "order": "segments", "requests": 6, "bare": 0.0},
        # A tuning step of four adapters trained side by side on a frozen projection.
        {"name": "adapter training, 4 adapters", "kind": "train", "dtype": "bf16", "T": 8192, "in": 4096, "out": 4096, "r": 16, "n": 4,
         "bias": False, "order": "segments", "requests": 16, "bare": 0.0, "weight_grad": False},
        # Tokens of seven adapters in no order, an odd token count, a rank that is no power of two.
        {"name": "adapter training, shuffled", "kind": "train", "dtype": "fp16", "T": 1537, "in": 1536, "out": 2880, "r": 24, "n": 7,
         "bias": True, "order": "shuffled", "requests": 200, "bare": 0.05, "weight_grad": False},
        # A small projection in 32 bits, everything trained, odd sizes.
        {"name": "adapter training, 32 bits", "kind": "train", "dtype": "fp32", "T": 301, "in": 200, "out": 123, "r": 5, "n": 3,
         "bias": True, "order": "segments", "requests": 4, "bare": 0.0, "weight_grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: mostly a multiple of 8 as layers have them, one in six any whole number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 1 / 6 else max(8, n // 8 * 8)


def draw(rng):
    kind = rng.choice(["mlp", "mlp", "moe", "adapter", "adapter", "train"])
    if kind in ("mlp", "moe"):
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"])
        E, d, F = _log(rng, 4, 128), _size(rng, 256, 4096), _size(rng, 128, 14336)
        layout = rng.choice(["plain", "glu_second", "glu_first", "interleaved"])
        width = 2 if layout == "plain" else 3
        most = 1.3e9 if dtype != "fp32" else 2e8
        F = max(64, min(F, int(most / (width * d * E)) // 8 * 8))
        c = {"kind": kind, "dtype": dtype, "T": _log(rng, 1, 64), "d": d, "F": F, "E": E, "k": rng.randint(1, min(8, E)),
             "layout": layout, "act": "silu" if layout != "plain" else rng.choice(["silu", "gelu"]), "bias": rng.random() < 0.4,
             "order": rng.choice(["out_in", "out_in", "in_out"])}
        if kind == "mlp":
            c["padded"] = rng.choice([0, 0, rng.randint(0, c["T"] - 1)])
        else:
            c["mode"] = rng.choice(["softmax_topk", "topk_softmax"])
        return c
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp16", "fp32"])
    T = _log(rng, 1, 8192) if kind == "adapter" else _log(rng, 64, 8192)
    if dtype == "fp32":
        T = min(T, 1024)
    wide = 4096 if dtype != "fp32" else 1024
    c = {"kind": kind, "dtype": dtype, "T": T, "in": _size(rng, 256, wide), "out": _size(rng, 256, wide), "r": _log(rng, 2, 64),
         "n": _log(rng, 1, 64), "bias": rng.random() < 0.4, "order": rng.choice(["segments", "segments", "shuffled"]),
         "requests": min(T, _log(rng, 1, 64)), "bare": rng.choice([0.0, 0.0, 0.1])}
    if kind == "train":
        c["weight_grad"] = rng.random() < 0.25
    return c


# ---- inputs -----------------------------------------------------------------------------------------


def _up_width(c):
    return c["F"] if c["layout"] == "plain" else 2 * c["F"]


def _matrices(g, dtype, E, rows, cols, order, scale):
    """(E, rows, cols) weights, a view: stored (E, cols, rows) for "out_in" (rows = inputs are contiguous), as they are for "in_out"."""
    if order == "out_in":
        return torch.empty(E, cols, rows, device="cuda", dtype=dtype).normal_(0.0, scale, generator=g).transpose(1, 2)
    return torch.empty(E, rows, cols, device="cuda", dtype=dtype).normal_(0.0, scale, generator=g)


def prepare(case, seed):
    c, dtype = case, DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, of=None):
        return torch.empty(*shape, device="cuda", dtype=of or dtype).normal_(0.0, scale, generator=g)

    s = {"case": c}
    if c["kind"] in ("mlp", "moe"):
        T, d, F, E, k = (c[n] for n in ("T", "d", "F", "E", "k"))
        s["x"] = normal(T, d)
        s["up"] = _matrices(g, dtype, E, d, _up_width(c), c["order"], d ** -0.5)
        s["down"] = _matrices(g, dtype, E, F, d, c["order"], F ** -0.5)
        s["up_b"] = normal(E, _up_width(c), scale=0.1) if c["bias"] else None
        s["down_b"] = normal(E, d, scale=0.1) if c["bias"] else None
        if c["kind"] == "moe":
            s["router"] = normal(E, d, scale=d ** -0.5)
            s["router_b"] = normal(E, scale=0.1) if c["bias"] else None
        else:
            score = torch.empty(T, E, device="cuda").normal_(generator=g)
            p, ids = torch.topk(torch.softmax(score, -1), k, dim=-1)
            if c["padded"]:
                ids[T - c["padded"]:] = -1
            s["gates"], s["ids"] = (p / p.sum(-1, keepdim=True)).to(dtype), ids
        return s
    T, n, r = c["T"], c["n"], c["r"]
    s["x"] = normal(T, c["in"])
    s["weight"] = normal(c["out"], c["in"], scale=c["in"] ** -0.5)
    s["a"] = normal(n, r, c["in"], scale=c["in"] ** -0.5)
    s["b"] = normal(n, c["out"], r, scale=r ** -0.5)
    s["bias"] = normal(c["out"], scale=0.1) if c["bias"] else None
    s["scaling"] = torch.empty(n, device="cuda").uniform_(0.25, 2.0, generator=g)
    # requests of ragged length, each with an adapter of its own choice (or none); "shuffled": their tokens interleaved
    cut = torch.sort(torch.randint(0, T, (c["requests"] - 1,), generator=g, device="cuda")).values
    request = torch.searchsorted(cut, torch.arange(T, device="cuda"), right=True)
    if c["order"] == "shuffled":
        request = request[torch.randperm(T, generator=g, device="cuda")]
    chosen = torch.randint(0, n, (c["requests"],), generator=g, device="cuda")
    chosen[torch.rand(c["requests"], generator=g, device="cuda") < c["bare"]] = -1
    s["ids"] = chosen[request]
    if c["kind"] == "train":
        s["dy"] = normal(T, c["out"])
        for name in ("x", "a", "b") + (("weight",) if c["weight_grad"] else ()) + (("bias",) if c["bias"] else ()):
            s[name].requires_grad_()
    return s


# ---- one pass ---------------------------------------------------------------------------------------


def run(state):
    c = state["case"]
    if own:
        return _run_own(c, state)
    with torch.no_grad():
        if c["kind"] == "mlp":
            return _plain_mlp(c, state, state["gates"].float(), state["ids"])
        if c["kind"] == "moe":
            return _plain_moe(c, state)
        return _plain_adapter(c, state)


def _run_own(c, s):
    import scattermoe_b200 as sm
    if c["kind"] == "mlp":
        return sm.few_token_mlp(s["x"], s["up"], s["down"], s["gates"], s["ids"], LAYOUTS[c["layout"]], ACTS[c["act"]],
                                up_biases=s["up_b"], down_biases=s["down_b"], alpha=ALPHA, limit=LIMIT)
    if c["kind"] == "moe":
        y, gates, ids = sm.few_token_moe(s["x"], s["router"], s["up"], s["down"], c["k"], LAYOUTS[c["layout"]], ACTS[c["act"]],
                                         mode=c["mode"], renormalize=True, router_bias=s["router_b"], up_biases=s["up_b"],
                                         down_biases=s["down_b"], alpha=ALPHA, limit=LIMIT)
        return {"y": y, "gates": gates, "ids": ids}
    y = sm.adapter_linear(s["x"], s["weight"], s["a"], s["b"], s["ids"], scaling=s["scaling"], bias=s["bias"])
    if c["kind"] == "adapter":
        return {"y": y}
    names = _trained(c)
    grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
    return {"y": y.detach(), **{"d_" + n: v for n, v in zip(names, grads)}}


def _trained(c):
    return ["x", "a", "b"] + (["weight"] if c["weight_grad"] else []) + (["bias"] if c["bias"] else [])


def _activate(c, u):
    if c["layout"] == "interleaved":
        gate, up = u[..., ::2].clamp(max=LIMIT), u[..., 1::2].clamp(-LIMIT, LIMIT)
        return (up + 1) * gate / (1 + torch.exp(-ALPHA * gate))
    if c["layout"] == "plain":
        gate, lin = u, 1.0
    else:
        first, second = u.chunk(2, -1)
        gate, lin = (first, second) if c["layout"] == "glu_first" else (second, first)
    if c["act"] == "silu":
        return gate / (1 + torch.exp(-gate)) * lin
    return 0.5 * gate * (1 + torch.erf(gate * 0.5 ** 0.5)) * lin


def _plain_mlp(c, s, gates, ids):
    """Few slots: the selected experts' matrices are gathered, one for each slot. Many: every expert on every token, weighted with
    the token's gate for it (zero where it was not selected)."""
    T, E, k = c["T"], c["E"], c["k"]
    live = (ids >= 0) & (ids < E)
    gates, safe = gates * live, ids.clamp(0, E - 1)
    x = s["x"].float()
    if T * k <= E:
        e = safe.flatten()
        u = torch.matmul(x.repeat_interleave(k, 0).unsqueeze(1), s["up"][e].float()).squeeze(1)
        u = u + s["up_b"][e].float() if c["bias"] else u
        y = torch.matmul(_activate(c, u).unsqueeze(1), s["down"][e].float()).squeeze(1)
        y = y + s["down_b"][e].float() if c["bias"] else y
        return (y.view(T, k, -1) * gates.unsqueeze(-1)).sum(1).to(s["x"].dtype)
    weight = torch.zeros(T, E, device="cuda").scatter_add_(1, safe, gates)
    u = torch.matmul(x, s["up"].float())
    u = u + s["up_b"].float().unsqueeze(1) if c["bias"] else u
    y = torch.matmul(_activate(c, u) * weight.t().unsqueeze(-1), s["down"].float()).sum(0)
    y = y + weight @ s["down_b"].float() if c["bias"] else y
    return y.to(s["x"].dtype)


def _plain_moe(c, s):
    z = s["x"].double() @ s["router"].double().t()
    z = (z + s["router_b"].double() if c["bias"] else z).float()
    top, ids = torch.topk(z, c["k"], dim=-1)
    w = torch.exp(top - top[:, :1])
    gates = w / w.sum(-1, keepdim=True)          # both modes: a softmax over the selected logits
    return {"y": _plain_mlp(c, s, gates, ids), "gates": gates, "ids": ids}


def _plain_adapter(c, s):
    n, r, dtype = c["n"], c["r"], s["x"].dtype
    x, w, a, b = (s[name].float() for name in ("x", "weight", "a", "b"))
    # every adapter on every token, (T, n r), masked to the token's own
    pick = (s["ids"].unsqueeze(1) == torch.arange(n, device="cuda")).float() * s["scaling"]
    pick = pick.repeat_interleave(r, 1)
    b_rows = b.transpose(1, 2).reshape(n * r, -1)
    h = (x @ a.reshape(n * r, -1).t()) * pick
    y = x @ w.t() + h @ b_rows
    y = y + s["bias"].float() if c["bias"] else y
    if c["kind"] == "adapter":
        return {"y": y.to(dtype)}
    dy = s["dy"].float()
    g = (dy @ b_rows.t()) * pick
    out = {"y": y, "d_x": dy @ w + g @ a.reshape(n * r, -1), "d_a": (g.t() @ x).view(n, r, -1),
           "d_b": (h.t() @ dy).view(n, r, -1).transpose(1, 2)}
    if c["weight_grad"]:
        out["d_weight"] = dy.t() @ x
    if c["bias"]:
        out["d_bias"] = dy.sum(0)
    return {name: v.to(dtype) for name, v in out.items()}


# ---- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] in ("mlp", "moe"):
        T, d, F, E, k = (c[n] for n in ("T", "d", "F", "E", "k"))
        T = T - c.get("padded", 0)
        active = E * (1 - (1 - k / E) ** T)                 # experts that occur, expected for even routing
        per_expert = d * _up_width(c) + F * d + ((_up_width(c) + d) if c["bias"] else 0)
        flops = 2.0 * T * k * d * (_up_width(c) + F)
        moved = active * per_expert * size + 2 * c["T"] * d * size + c["T"] * k * (8 + size)
        if c["kind"] == "moe":
            flops += 2.0 * T * E * d
            moved += E * d * size
        return {"bytes": moved, "flops": flops}
    T, i, o, r, n = c["T"], c["in"], c["out"], c["r"], c["n"]
    used = n * (1 - (1 - 1 / n) ** c["requests"])           # adapters that occur
    flops = 2.0 * T * i * o + 2.0 * T * r * (i + o)
    moved = size * (i * o + used * r * (i + o) + T * (i + o)) + 8 * T
    if c["kind"] == "train":
        flops += 2.0 * T * i * o * (2 if c["weight_grad"] else 1) + 6.0 * T * r * (i + o) - 2.0 * T * r * i
        moved += size * (T * (i + o) + n * r * (i + o) + (i * o if c["weight_grad"] else 0))
    return {"bytes": moved, "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] in ("mlp", "moe"):
            return _exact_layer(case, s)
        return _exact_adapter(case, s)


def _exact_act(c, u):
    f = u.shape[-1] // 2
    if c["layout"] == "interleaved":
        g = torch.minimum(u[:, 0::2], torch.tensor(LIMIT, device="cuda", dtype=torch.float64))
        v = torch.clamp(u[:, 1::2], -LIMIT, LIMIT)
        return (v + 1.0) * (g * torch.sigmoid(ALPHA * g))
    phi = (lambda z: z * torch.sigmoid(z)) if c["act"] == "silu" else (lambda z: z * 0.5 * torch.erfc(-z / math.sqrt(2.0)))
    if c["layout"] == "plain":
        return phi(u)
    return phi(u[:, :f]) * u[:, f:] if c["layout"] == "glu_first" else phi(u[:, f:]) * u[:, :f]


def _exact_layer(c, s):
    x = s["x"].double()
    if c["kind"] == "moe":
        z = torch.einsum("td,ed->te", x, s["router"].double())
        z = z + s["router_b"].double() if c["bias"] else z
        order = torch.argsort(z, dim=1, descending=True, stable=True)[:, :c["k"]]
        gates, ids = torch.softmax(torch.gather(z, 1, order), 1), order
    else:
        gates, ids = s["gates"].double(), s["ids"]
    y = torch.zeros(c["T"], c["d"], device="cuda", dtype=torch.float64)
    for e in range(c["E"]):                                  # expert by expert, on the rows that chose it
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if not t.numel():
            continue
        u = x[t] @ s["up"][e].double()
        u = u + s["up_b"][e].double() if c["bias"] else u
        v = _exact_act(c, u) @ s["down"][e].double()
        v = v + s["down_b"][e].double() if c["bias"] else v
        y.index_add_(0, t, v * gates[t, j].unsqueeze(1))
    return y if c["kind"] == "mlp" else {"y": y, "gates": gates, "ids": ids}


def _exact_adapter(c, s):
    x, w = s["x"].double(), s["weight"].double()
    y = x @ w.t() + (s["bias"].double() if c["bias"] else 0.0)
    train = c["kind"] == "train"
    if train:
        dy = s["dy"].double()
        dx, da, db = dy @ w, torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
    for e in range(c["n"]):                                  # adapter by adapter, on its own rows
        t = torch.nonzero(s["ids"] == e).flatten()
        if not t.numel():
            continue
        a, b, f = s["a"][e].double(), s["b"][e].double(), s["scaling"][e].double()
        y[t] += f * (x[t] @ a.t()) @ b.t()
        if train:
            dx[t] += f * (dy[t] @ b) @ a
            da[e] = f * (dy[t] @ b).t() @ x[t]
            db[e] = f * dy[t].t() @ (x[t] @ a.t())
    if not train:
        return {"y": y}
    out = {"y": y, "d_x": dx, "d_a": da, "d_b": db}
    if c["weight_grad"]:
        out["d_weight"] = dy.t() @ x
    if c["bias"]:
        out["d_bias"] = dy.sum(0)
    return out
