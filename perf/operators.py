"""Cases that time the 8-bit operators of webllm_b200: the row quantiser, the dense product with a scale per token and
per channel, the expert router, and the products grouped by expert.

`run` computes a case in plain torch operations, or through the library's entry points where `own` is set.

  quantize   v -> (q, s): s = max|v| / 127 of each row, q = the integers nearest v / s
  product    y[n][m] = s[n] t[m] sum_k q[n][k] w[m][k], x quantised per token in the pass
  route      the k largest logits of each token, their weights, and the slots sorted by expert
  experts    each token's k experts: the first product of a feed-forward block ("up": rows of x to rows per slot), or
             its last ("down": silu(gate) * up of each slot, the expert's product, the weighted sum over a token's slots)
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token's hidden state ahead of a decode projection
        {"name": "quantize_token", "op": "quantize", "rows": 1, "K": 4096, "x": "f32"},
        # a long prompt's feed-forward activations
        {"name": "quantize_prompt", "op": "quantize", "rows": 8192, "K": 14336, "x": "bf16"},
        # decode of one sequence: an FFN gate projection, f32 activations as the framework's other ops have them
        {"name": "product_token", "op": "product", "N": 1, "K": 4096, "M": 14336, "x": "f32", "y": "f32"},
        # an odd number of sequences decoding together
        {"name": "product_batch", "op": "product", "N": 33, "K": 2304, "M": 9216, "x": "f16", "y": "f16"},
        # a prompt of 512 tokens through an FFN projection
        {"name": "product_prompt", "op": "product", "N": 512, "K": 4096, "M": 14336, "x": "bf16", "y": "bf16"},
        # a long prompt through the down projection
        {"name": "product_long", "op": "product", "N": 4096, "K": 14336, "M": 4096, "x": "f32", "y": "f32"},
        # one token's router, 64 experts
        {"name": "route_token", "op": "route", "T": 1, "E": 64, "k": 8, "score": "softmax", "normalize": True},
        # a long prompt's router, 128 experts
        {"name": "route_prompt", "op": "route", "T": 8192, "E": 128, "k": 8, "score": "softmax", "normalize": True},
        # one token's gate and up projections in its 8 experts
        {"name": "experts_token", "op": "experts", "part": "up", "T": 1, "E": 64, "k": 8, "K": 2048, "M": 2048, "x": "f32", "y": "f32"},
        # an odd number of sequences decoding: their experts' down projections and the sum over experts
        {"name": "experts_batch", "op": "experts", "part": "down", "T": 37, "E": 60, "k": 4, "K": 1152, "M": 2304, "x": "bf16", "y": "bf16"},
        # a prompt of 512 tokens: gate and up
        {"name": "experts_prompt", "op": "experts", "part": "up", "T": 512, "E": 64, "k": 8, "K": 2048, "M": 2048, "x": "bf16", "y": "bf16"},
        # a long prompt: down and the sum over experts
        {"name": "experts_long", "op": "experts", "part": "down", "T": 4096, "E": 128, "k": 8, "K": 1536, "M": 4096, "x": "bf16", "y": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A row length or a channel count: a multiple of 64 as model sizes are, or any number."""
    v = _log(rng, lo, hi)
    return v if rng.random() < 0.3 else max(64, v // 64 * 64)


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "route", "experts", "experts", "experts"])
    t = rng.choice(list(TYPES))
    if op == "quantize":
        K = _width(rng, 64, 16384)
        return {"op": op, "rows": _log(rng, 1, min(8192, 8192 * 14336 // K)), "K": K, "x": t}
    if op == "product":
        K, M = _width(rng, 256, 14336), _width(rng, 256, 14336)
        return {"op": op, "N": _log(rng, 1, min(4096, 4096 * 14336 * 4096 // (K * M))), "K": K, "M": M, "x": t, "y": t}
    k = rng.choice([1, 2, 4, 6, 8])
    E = rng.choice([8, 16, 60, 64, 96, 128, 256])
    if op == "route":
        return {"op": op, "T": _log(rng, 1, 8192), "E": E, "k": k, "score": rng.choice(["softmax", "sigmoid"]), "normalize": rng.random() < 0.5}
    part = rng.choice(["up", "down"])
    K, M = _width(rng, 256, 2048), _width(rng, 256, 4096)
    E = min(E, 128 * 1536 * 4096 // (K * M))
    t = "bf16" if part == "down" else t
    return {"op": op, "part": part, "T": _log(rng, 1, min(4096, 4096 * 8 * 1536 * 4096 // (K * M * k))), "E": max(E, 8), "k": k, "K": K, "M": M, "x": t, "y": t}


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "quantize":
        n = case["rows"] * case["K"]
        return {"bytes": n * (size[case["x"]] + 1) + 4 * case["rows"], "flops": 3 * n}
    if case["op"] == "product":
        N, K, M = case["N"], case["K"], case["M"]
        return {"bytes": N * K * size[case["x"]] + M * K + 4 * M + N * M * size[case["y"]], "flops": 2 * N * K * M}
    T, E, k = case["T"], case["E"], case["k"]
    if case["op"] == "route":
        return {"bytes": 4 * T * E + 12 * T * k + 4 * (E + 1), "flops": 4 * T * E}
    K, M = case["K"], case["M"]
    used = E * (1 - (1 - k / E) ** T)  # the experts that T tokens are expected to reach
    rows_in = T * K if case["part"] == "up" else T * k * 2 * K
    rows_out = T * k * M if case["part"] == "up" else T * M
    return {"bytes": rows_in * size[case["x"]] + used * M * (K + 4) + rows_out * size[case["y"]] + 12 * T * k, "flops": 2 * T * k * K * M}


# ---------------------------------------------------------------- inputs


def _up16(n):
    return (n + 15) // 16 * 16


def _rows8(gen, rows, K):
    """int8 rows with one scale each, as a trained weight quantised per channel has them; rows are 16-byte multiples apart."""
    q = torch.zeros(rows, _up16(K), dtype=torch.int8, device="cuda")
    s = torch.empty(rows, device="cuda")
    step = max(1, (1 << 28) // K)
    for r in range(0, rows, step):
        v = torch.randn(min(step, rows - r), K, device="cuda", generator=gen)
        a = v.abs().amax(1, keepdim=True)
        q[r : r + step, :K] = (v * (127.0 / a)).round_().to(torch.int8)
        s[r : r + step] = a[:, 0] * (0.02 / 127.0)
    return q, s


def _acts(gen, rows, K, t):
    """Activations: normal values, a few channels some times larger, rows of different size."""
    x = torch.randn(rows, K, device="cuda", generator=gen)
    x[:, torch.randint(0, K, (max(1, K // 512),), device="cuda", generator=gen)] *= 8
    x *= 0.25 + 1.5 * torch.rand(rows, 1, device="cuda", generator=gen)
    return x.to(TYPES[t])


def _logits(gen, T, E):
    """Router logits: some experts are liked better than others."""
    return torch.randn(T, E, device="cuda", generator=gen) + 0.5 * torch.randn(E, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    empty = lambda *shape, t=torch.float32: torch.empty(*shape, dtype=t, device="cuda")  # noqa: E731
    if case["op"] == "quantize":
        n, K = case["rows"], case["K"]
        s |= {"x_": _acts(gen, n, K, case["x"]), "q": empty(n, _up16(K), t=torch.int8), "s": empty(n)}
    elif case["op"] == "product":
        N, K, M = case["N"], case["K"], case["M"]
        w, t = _rows8(gen, M, K)
        s |= {"x_": _acts(gen, N, K, case["x"]), "w": w, "t": t, "q": empty(N, _up16(K), t=torch.int8), "s": empty(N), "y_": empty(N, M, t=TYPES[case["y"]])}
    elif case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        s |= {"logits": _logits(gen, T, E), "ids": empty(T, k, t=torch.int32), "weights": empty(T, k), "offsets": empty(E + 1, t=torch.int32), "order": empty(T * k, t=torch.int32)}
    else:
        T, E, k, K, M = (case[n] for n in ("T", "E", "k", "K", "M"))
        w, t = _rows8(gen, E * M, K)
        top, ids = _logits(gen, T, E).topk(k, 1)
        count = torch.bincount(ids.flatten(), minlength=E)
        rows = T if case["part"] == "up" else T * k
        x = _acts(gen, rows, K if case["part"] == "up" else 2 * K, case["x"])
        # the routing that an earlier step made: experts and weights of each token, and the slots in the order of their expert
        s |= {
            "x_": x, "w": w.view(E, M, -1), "t": t.view(E, M), "ids": ids.to(torch.int32), "weights": top.softmax(1),
            "order": ids.flatten().sort(stable=True).indices.to(torch.int32), "offsets": torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32), "capacity": int(count.max()),
            "q": empty(rows, _up16(K), t=torch.int8), "s": empty(rows), "y_": empty(T * k, M, t=TYPES[case["y"]] if case["part"] == "up" else torch.float16),
        }
        if case["part"] == "down":
            s["sum"] = empty(T, M, t=TYPES[case["y"]])
    return s


# ---------------------------------------------------------------- plain forms


def _quantize(v):
    """(q, s) of the rows of v. The quotients are taken in 64 bits: those next to a half decide a whole number."""
    s = (v.abs().amax(1).double() / 127).float()
    q = torch.where(s[:, None] > 0, v.double() / s[:, None].double(), 0.0).round().clamp(-127, 127)
    return q.float(), s


def _route(st):
    l, E, k = st["logits"].float(), st["E"], st["k"]
    ids = l.sort(dim=1, descending=True, stable=True).indices[:, :k]
    if st["score"] == "softmax":
        p = (l - l.amax(1, keepdim=True)).exp()
        w = p.gather(1, ids)
        w = w / (w if st["normalize"] else p).sum(1, keepdim=True)
    else:
        w = 1 / (1 + (-l.gather(1, ids)).exp())
        w = w / w.sum(1, keepdim=True) if st["normalize"] else w
    flat = ids.flatten()
    count = (flat[:, None] == torch.arange(E, device=l.device)).sum(0)
    offsets = torch.cat([count.new_zeros(1), count.cumsum(0)])
    return [ids.to(torch.int32), w, offsets.to(torch.int32), flat.sort(stable=True).indices.to(torch.int32)]


def _experts(st):
    T, E, k, K, M = (st[n] for n in ("T", "E", "k", "K", "M"))
    if st["part"] == "up":
        q, s = _quantize(st["x_"].float())
        q, s = q.repeat_interleave(k, 0), s.repeat_interleave(k, 0)
    else:
        g, u = st["x_"].double().chunk(2, 1)
        q, s = _quantize(g / (1 + (-g).exp()) * u)
    slot = st["ids"].flatten().long()
    if T * k <= E:
        y = (st["w"][slot, :, :K].float() @ q[:, :, None])[:, :, 0]
    else:  # every expert's rows side by side, to the most that one has
        order = st["order"].long()
        at = torch.arange(T * k, device=slot.device) - st["offsets"].long()[slot[order]]
        wide = q.new_zeros(E, st["capacity"], K)
        wide[slot[order], at] = q[order]
        y = q.new_empty(T * k, M)
        y[order] = (wide @ st["w"][:, :, :K].float().transpose(1, 2))[slot[order], at]
    y = y * s[:, None] * st["t"][slot]
    if st["part"] == "down":
        y = (y.view(T, k, M) * st["weights"][:, :, None]).sum(1)
    return y.to(TYPES[st["y"]])


def _plain(st):
    if st["op"] == "quantize":
        q, s = _quantize(st["x_"].float())
        return [q.to(torch.int8), s]
    if st["op"] == "product":
        q, s = _quantize(st["x_"].float())
        return (q @ st["w"][:, : st["K"]].float().t() * s[:, None] * st["t"]).to(TYPES[st["y"]])
    return _route(st) if st["op"] == "route" else _experts(st)


# ---------------------------------------------------------------- the library's operators


def _own(st):
    from webllm_b200 import jsep

    jsep.install_jsep_callbacks(torch.cuda.current_device())
    stream = torch.cuda.current_stream().cuda_stream or jsep.STREAM_LEGACY
    types = {"f32": jsep.GGML_TYPE_F32, "f16": jsep.GGML_TYPE_F16, "bf16": jsep.GGML_TYPE_BF16}
    if st["op"] == "route":
        T, E, k = st["T"], st["E"], st["k"]
        ids, weights, offsets, order = st["ids"], st["weights"], st["offsets"], st["order"]
        jsep.moe_route(st["logits"].data_ptr(), E, T, E, k, jsep.MOE_SOFTMAX if st["score"] == "softmax" else jsep.MOE_SIGMOID, st["normalize"], 1.0,
                       ids.data_ptr(), weights.data_ptr(), stream=stream)
        jsep.moe_plan(ids.data_ptr(), T, k, E, offsets.data_ptr(), order.data_ptr(), stream=stream)
        return [ids, weights, offsets, order]
    x, q, s, K = st["x_"], st["q"], st["s"], st["K"]
    tx, rows, pitch = types[st["x"]], x.shape[0], q.shape[1]
    if st.get("part") == "down":  # gate and up are the halves of each row
        jsep.quantize_i8(tx, x.data_ptr(), 2 * K, rows, K, q.data_ptr(), pitch, s.data_ptr(), glu=jsep.GLU_SWIGLU, up_ptr=x.data_ptr() + K * x.element_size(), up_stride=2 * K, stream=stream)
    else:
        jsep.quantize_i8(tx, x.data_ptr(), K, rows, K, q.data_ptr(), pitch, s.data_ptr(), stream=stream)
    if st["op"] == "quantize":
        return [q[:, :K], s]
    w, t, y, M = st["w"], st["t"], st["y_"], st["M"]
    if st["op"] == "product":
        jsep.mul_mat_i8(w.data_ptr(), pitch, t.data_ptr(), q.data_ptr(), pitch, s.data_ptr(), types[st["y"]], y.data_ptr(), M, M, K, rows, stream=stream)
        return y
    T, k, up = st["T"], st["k"], st["part"] == "up"
    tz = types[st["y"]]
    if not up:  # the slots' rows stay in 32 bits ahead of their sum: in 16 they would be rounded twice, and f16 ends at 65504
        y, tz = y.new_empty(y.shape, dtype=torch.float32), jsep.GGML_TYPE_F32
    jsep.mul_mat_id_i8(w.data_ptr(), pitch, M * pitch, t.data_ptr(), q.data_ptr(), pitch, s.data_ptr(), not up, st["offsets"].data_ptr(), st["order"].data_ptr(),
                       tz, y.data_ptr(), M, M, K, st["E"], T, k, stream=stream)
    if up:
        return y
    jsep.moe_combine(tz, y.data_ptr(), M, st["weights"].data_ptr(), types[st["y"]], st["sum"].data_ptr(), M, T, k, M, stream=stream)
    return st["sum"]


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    st = prepare(case, seed)

    def rows8(v):
        s = (v.abs().max(dim=-1).values / 127.0).to(torch.float32).to(torch.float64)
        q = torch.zeros_like(v)
        live = s > 0
        q[live] = torch.clamp(torch.round(v[live] / s[live].unsqueeze(-1)), -127.0, 127.0)
        return q, s

    if case["op"] == "quantize":
        q, s = rows8(st["x_"].double())
        return [q.to(torch.int8), s]
    if case["op"] == "product":
        q, s = rows8(st["x_"].double())
        return torch.einsum("nk,mk->nm", q, st["w"][:, : case["K"]].double()) * torch.outer(s, st["t"].double())
    if case["op"] == "route":
        l = st["logits"].double()
        left, ids = l.clone(), []
        for _ in range(case["k"]):
            best = (left == left.max(dim=1, keepdim=True).values).double().argmax(dim=1)  # the first of the largest
            ids.append(best)
            left[torch.arange(len(l), device=l.device), best] = -math.inf
        ids = torch.stack(ids, 1)
        p = torch.softmax(l, 1) if case["score"] == "softmax" else torch.sigmoid(l)
        w = torch.gather(p, 1, ids)
        if case["normalize"]:
            w = w / w.sum(1, keepdim=True)
        slots = [(ids.flatten() == e).nonzero().flatten() for e in range(case["E"])]
        offsets = torch.tensor([0] + [len(v) for v in slots], device=l.device).cumsum(0)
        return [ids.to(torch.int32), w, offsets.to(torch.int32), torch.cat(slots).to(torch.int32)]
    T, E, k, K, M = (case[n] for n in ("T", "E", "k", "K", "M"))
    x = st["x_"].double()
    if case["part"] == "down":
        x = torch.nn.functional.silu(x[:, :K]) * x[:, K:]
    q, s = rows8(x)
    ids = st["ids"].flatten()
    y = torch.zeros(T * k, M, dtype=torch.float64, device="cuda")
    for e in range(E):
        at = (ids == e).nonzero().flatten()
        row = at // k if case["part"] == "up" else at
        y[at] = torch.einsum("nk,mk->nm", q[row], st["w"][e, :, :K].double()) * torch.outer(s[row], st["t"][e].double())
    return torch.einsum("tjm,tj->tm", y.view(T, k, M), st["weights"].double()) if case["part"] == "down" else y
