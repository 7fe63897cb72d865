"""Operators of a block that is trained or served in plain rows, as measurable cases.

  route       a token's choice of experts from its router logits, and its gates
                s = softmax(l) or sigmoid(l); the k experts of largest s + b (ties:
                the lowest index), best first, of the expert groups whose best
                one or two s + b sum to most;
                gate_j = scale s_j / (renormalize ? sum over the chosen s : 1)
              with the rows in expert order that the ragged products take
              (offsets, the token of each row, the row of each choice), and the
              gradient of the logits
  norm        s = x + residual, y = s / sqrt(mean(s^2) + eps) w, y in the values' type
              or in 8 bits with scales, and the gradients of x and w
  product     z = W_g x + b_g, y = act(z) * factor + residual in one call, z kept for
              the backward where it is asked for; the gradients of z, the factor
              and the biases
  activation  y = act(gate) * up with gate and up kept in 8 bits, and the gradients
              from what was kept, y made again on the way
  pack        rows into 8 bits and back

8 bits: every scale_columns columns of a row share scale = max|v| / 127 (int8) or
/ 448 (e4m3) in float32; int8 codes are v / scale to the nearest, halves away from
zero, e4m3 codes the float32 quotient to the nearest, halves to even.

Shapes are those the benchmark and the tests run: d=1024 E=16 k=2 h=2048;
d=1024 E=64 k=6 h=512; d=2048 E=128 k=8 h=768; d=2048 E=64 k=4 h=1024; d=256
E=8 k=2 h=512; and the ragged d=1000 E=14 k=3 h=1201."""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SHAPES = {
    "small": dict(d=256, h=512, E=8, k=2, zipf=0.0),
    "wide": dict(d=1024, h=2048, E=16, k=2, zipf=0.0),
    "many": dict(d=1024, h=512, E=64, k=6, zipf=0.0),
    "skewed": dict(d=2048, h=768, E=128, k=8, zipf=0.6),
    "block": dict(d=2048, h=1024, E=64, k=4, zipf=0.0),
    "ragged": dict(d=1000, h=1201, E=14, k=3, zipf=0.3),
}
EPSILON = 1e-6


def _route(tokens, experts, k, values, scores="softmax", bias=False, groups=1, chosen_groups=1, best=1, renormalize=True,
           scale=1.0, training=False):
    return dict(kind="route", values=values, tokens=tokens, experts=experts, k=k, scores=scores, bias=bias, groups=groups,
                chosen_groups=chosen_groups, best=best, renormalize=renormalize, scale=scale, training=training)


def _norm(rows, columns, values, codes="none", scale_columns=128, training=False):
    return dict(kind="norm", values=values, rows=rows, columns=columns, codes=codes, scale_columns=scale_columns,
                training=training)


def _product(rows, groups, inputs, outputs, values, activation="none", bias=False, factor=False, residual=False, zipf=0.0,
             training=False):
    return dict(kind="product", values=values, rows=rows, groups=groups, inputs=inputs, outputs=outputs,
                activation=activation, bias=bias, factor=factor, residual=residual, zipf=zipf, training=training)


def _activation(rows, columns, values, activation, codes, scale_columns, limit=0.0):
    return dict(kind="activation", values=values, rows=rows, columns=columns, activation=activation, codes=codes,
                scale_columns=scale_columns, limit=limit)


def _pack(rows, columns, values, codes, scale_columns):
    return dict(kind="pack", values=values, rows=rows, columns=columns, codes=codes, scale_columns=scale_columns)


def listed():
    cases = {
        # a decode batch of 32 sequences over 64 experts
        "route_f32_decode": _route(32, 64, 6, "f32"),
        # a long prompt over 128 experts in eight groups, balanced by biases
        "route_bf16_prefill": _route(16384, 128, 8, "bf16", scores="sigmoid", bias=True, groups=8, chosen_groups=4, best=2,
                                     scale=2.5),
        # a router's training step: the choice and the logits' gradients
        "route_f32_training": _route(8192, 64, 4, "f32", renormalize=False, training=True),
        # one generated token, normed into 8 bits
        "norm_bf16_t1": _norm(1, 2048, "bf16", codes="e4m3"),
        # a training batch: the residual's sum, the norm, and its gradients
        "norm_bf16_training": _norm(8192, 2048, "bf16", training=True),
        # full precision, odd widths
        "norm_f32_ragged": _norm(2331, 1201, "f32", training=True),
        # the gate of a dense SwiGLU over a decode batch, times the up projection's rows
        "product_bf16_decode": _product(32, 1, 1024, 2048, "bf16", activation="silu", bias=True, factor=True),
        # the experts' gates of a training batch, what their backward needs kept, and that backward
        "product_bf16_training": _product(16384, 16, 1024, 2048, "bf16", activation="silu", bias=True, factor=True,
                                          training=True),
        # a dense down projection of a prompt onto the residual stream
        "product_f16_residual": _product(8192, 1, 1024, 2048, "f16", bias=True, residual=True),
        # the experts' SwiGLU of a training batch with 8-bit checkpoints
        "activation_bf16_training": _activation(16384, 2048, "bf16", "silu", "int8", 128),
        # odd widths and small blocks, full precision
        "activation_f32_ragged": _activation(2331, 1201, "f32", "gelu", "e4m3", 32, limit=10.0),
        # a layer's inputs kept in the library's Int8 rows
        "pack_f16": _pack(8192, 2048, "f16", "int8", 16),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["route", "route", "norm", "norm", "product", "product", "activation", "pack"])
    values = rng.choice(["bf16", "bf16", "f16", "f32"])
    shape = SHAPES[rng.choice(list(SHAPES))]
    if kind == "route":
        experts = rng.choice([shape["E"], shape["E"], 256])
        groups = rng.choice([g for g in (1, 1, 2, 4, 7, 8) if experts % g == 0])
        chosen = rng.randint(max(1, groups // 2), groups)
        k = min(rng.choice([1, shape["k"], shape["k"], 8]), experts // groups * chosen)
        return _route(log_int(1, 16384), experts, k, values, scores=rng.choice(["softmax", "sigmoid"]),
                      bias=rng.random() < 0.5, groups=groups, chosen_groups=chosen,
                      best=rng.choice([1, 2]) if experts // groups > 1 else 1, renormalize=rng.random() < 0.6,
                      scale=rng.choice([1.0, 2.5]), training=rng.random() < 0.4)
    if kind == "norm":
        codes = rng.choice(["none", "none", "int8", "e4m3"]) if values != "f32" else "none"
        return _norm(log_int(1, 4096 if values == "f32" else 8192), rng.choice([shape["d"], shape["h"], log_int(16, 4096)]), values, codes=codes,
                     scale_columns=rng.choice([16, 32, 64, 128, 0]), training=codes == "none" and rng.random() < 0.6)
    if kind == "product":
        sides = [shape["d"], shape["h"]]
        rng.shuffle(sides)
        groups = rng.choice([1, 1, shape["E"]])
        rows = log_int(1, 2048 if values == "f32" else 16384)
        return _product(rows, groups, sides[0], sides[1], values, activation=rng.choice(["none", "silu", "gelu", "relu"]),
                        bias=rng.random() < 0.7, factor=rng.random() < 0.5, residual=rng.random() < 0.4,
                        zipf=shape["zipf"] if groups > 1 else 0.0, training=rng.random() < 0.4)
    rows = log_int(1, 8192 if values == "f32" else 16384)
    columns = rng.choice([shape["d"], shape["h"], log_int(8, 2048)])
    codes, scale_columns = rng.choice(["int8", "e4m3"]), rng.choice([16, 32, 64, 128])
    if kind == "activation":
        return _activation(rows, columns, values, rng.choice(["silu", "silu", "gelu", "relu"]), codes, scale_columns,
                           limit=rng.choice([0.0, 0.0, 10.0]))
    return _pack(rows, columns, values, codes, rng.choice([scale_columns, 0]))


# --------------------------------------------------------------------------
# inputs, from the seed alone
# --------------------------------------------------------------------------

def _offsets(case, seed):
    g = np.random.default_rng([seed, case["rows"], 78])
    p = 1.0 / np.arange(1, case["groups"] + 1) ** case["zipf"]
    sizes = g.multinomial(case["rows"], g.permutation(p / p.sum()))
    return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)


def _made(case, seed):
    """The arrays of the case on the GPU."""
    t, kind = TYPES[case["values"]], case["kind"]
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + case.get("rows", case.get("tokens", 0)))

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype or t)

    if kind == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        return dict(logits=normal(T, E, scale=1.5),
                    bias=normal(E, scale=0.1, dtype=torch.float32) if case["bias"] else None,
                    dgates=normal(T, k, dtype=torch.float32))
    R = case["rows"]
    if kind == "norm":
        C = case["columns"]
        return dict(x=normal(R, C), residual=normal(R, C, scale=2.0), w=(normal(C, scale=0.2, dtype=torch.float32) + 1).to(t),
                    dy=normal(R, C), dsum=normal(R, C))
    if kind == "product":
        K, N, G = case["inputs"], case["outputs"], case["groups"]
        offsets = _offsets(case, seed)
        return dict(offsets=torch.from_numpy(offsets).cuda() if G > 1 else None, most=int(np.diff(offsets).max()),
                    x=normal(R, K), w=normal(G, N, K, scale=K ** -0.5),
                    b=normal(G, N, scale=0.5) if case["bias"] else None,
                    factor=normal(R, N) if case["factor"] else None,
                    residual=normal(R, N) if case["residual"] else None, dy=normal(R, N))
    if kind == "activation":
        C = case["columns"]
        return dict(gate=normal(R, C, scale=2.0), up=normal(R, C, scale=2.0), dy=normal(R, C))
    return dict(x=normal(R, case["columns"], scale=3.0))


_context = None


def prepare(case, seed):
    s = _made(case, seed)
    s["case"] = case
    if own:
        s.update(_plan(case))
    return s


def _plan(case):
    """What a program keeps between calls: descriptions, output buffers, workspaces."""
    import gotransformers_amd as gt

    global _context
    if _context is None:
        _context = gt.Context(0)
    t, kind = TYPES[case["values"]], case["kind"]
    values = {"f32": gt.VALUES_FLOAT32, "bf16": gt.VALUES_BFLOAT16, "f16": gt.VALUES_FLOAT16}[case["values"]]

    def empty(*shape, dtype=t):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    if kind == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        d = gt.route_desc(values, T, E, k, expert_groups=case["groups"], chosen_groups=case["chosen_groups"],
                          group_best=case["best"], renormalize=case["renormalize"], scale=case["scale"],
                          scores=gt.SCORES_SIGMOID if case["scores"] == "sigmoid" else gt.SCORES_SOFTMAX)
        return dict(desc=d, chosen=empty(T, k, dtype=torch.int32), gates=empty(T, k, dtype=torch.float32),
                    offsets=empty(E + 1, dtype=torch.int32), rows=empty(T * k, dtype=torch.int32),
                    places=empty(T, k, dtype=torch.int32), dlogits=empty(T, E),
                    workspace=empty(gt.route_workspace_bytes(d), dtype=torch.uint8))
    R = case["rows"]
    if kind == "product":
        G, N = case["groups"], case["outputs"]
        d = gt.grouped_desc(values, G, R, case["inputs"], N)
        act = {"none": gt.ACTIVATION_NONE, "silu": gt.ACTIVATION_SILU, "gelu": gt.ACTIVATION_GELU,
               "relu": gt.ACTIVATION_RELU}[case["activation"]]
        return dict(desc=d, activation=act, act_desc=gt.activation_desc(values, R, N, act), y=empty(R, N), z=empty(R, N),
                    dz=empty(R, N), dfactor=empty(R, N), db=empty(G, N),
                    workspace=empty(gt.grouped_bias_workspace_bytes(d), dtype=torch.uint8))
    C = case["columns"]
    codes = {"none": gt.CODES_NONE, "int8": gt.CODES_INT8, "e4m3": gt.CODES_E4M3}[case["codes"]]
    blocks = -(-C // (case["scale_columns"] or C))

    def packed():
        return empty(R, C, dtype=torch.uint8), empty(R, blocks, dtype=torch.float32)

    if kind == "norm":
        d = gt.norm_desc(values, R, C, epsilon=EPSILON, codes=codes, scale_columns=case["scale_columns"])
        p = dict(desc=d, sums=empty(R, C), y=empty(R, C), dx=empty(R, C), dw=empty(C, dtype=torch.float32),
                 workspace=empty(gt.norm_workspace_bytes(d), dtype=torch.uint8))
        if case["codes"] != "none":
            p["codes"], p["scales"] = packed()
            p["packed_desc"] = gt.packed_desc(values, R, C, codes, case["scale_columns"])
        return p
    if kind == "activation":
        act = {"silu": gt.ACTIVATION_SILU, "gelu": gt.ACTIVATION_GELU, "relu": gt.ACTIVATION_RELU}[case["activation"]]
        p = dict(desc=gt.activation_desc(values, R, C, act, limit=case["limit"], codes=codes,
                                         scale_columns=case["scale_columns"]),
                 y=empty(R, C), again=empty(R, C), dgate=empty(R, C), dup=empty(R, C))
        (p["gate_codes"], p["gate_scales"]), (p["up_codes"], p["up_scales"]) = packed(), packed()
        return p
    p = dict(desc=gt.packed_desc(values, R, C, codes, case["scale_columns"]), y=empty(R, C))
    p["codes"], p["scales"] = packed()
    return p


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import gotransformers_amd as gt

    case, ctx, d = s["case"], _context, s["desc"]
    stream = torch.cuda.current_stream().cuda_stream
    kind = case["kind"]

    def p(name):
        v = s.get(name)
        return None if v is None else v.data_ptr()

    if kind == "route":
        gt.route_forward(ctx, d, p("logits"), p("bias"), p("chosen"), p("gates"), p("offsets"), p("rows"), p("places"),
                         p("workspace"), stream)
        out = {n: s[n] for n in ("chosen", "gates", "offsets", "rows", "places")}
        if case["training"]:
            gt.route_gradient(ctx, d, p("logits"), p("chosen"), p("dgates"), p("dlogits"), stream)
            out["dlogits"] = s["dlogits"]
        return out
    if kind == "norm":
        gt.norm_forward(ctx, d, p("x"), p("residual"), p("w"), p("sums"), None if "codes" in s else p("y"), p("codes"),
                        p("scales"), stream)
        if "codes" in s:
            gt.unpack_rows(ctx, s["packed_desc"], p("codes"), p("scales"), p("y"), stream)
        out = {"sums": s["sums"], "y": s["y"]}
        if case["training"]:
            gt.norm_gradient(ctx, d, p("dy"), p("sums"), p("w"), p("dsum"), p("dx"), p("dw"), gt.VALUES_FLOAT32, False,
                             p("workspace"), stream)
            out.update(dx=s["dx"], dw=s["dw"])
        return out
    if kind == "product":
        e = gt.epilogue(s["activation"], biases_ptr=p("b"), factors_ptr=p("factor"), residuals_ptr=p("residual"),
                        products_ptr=p("z") if case["training"] else None, width=case["outputs"])
        gt.grouped_fused_forward(ctx, d, e, p("offsets"), p("x"), p("w"), p("y"), stream)
        out = {"y": s["y"]}
        if case["training"]:
            out["z"] = s["z"]
            gt.activation_gradient(ctx, s["act_desc"], p("dy"), p("z"), None, p("factor"), None, p("dz"),
                                   p("dfactor") if case["factor"] else None, None, stream)
            out["dz"] = s["dz"]
            if case["factor"]:
                out["dfactor"] = s["dfactor"]
            if case["bias"]:
                gt.grouped_bias_gradient(ctx, d, p("offsets"), p("dz"), p("db"), d.values, False, p("workspace"), stream)
                out["db"] = s["db"]
        return out
    if kind == "activation":
        gt.activation_forward(ctx, d, p("gate"), p("up"), p("y"), p("gate_codes"), p("gate_scales"), p("up_codes"),
                              p("up_scales"), stream)
        gt.activation_gradient(ctx, d, p("dy"), p("gate_codes"), p("gate_scales"), p("up_codes"), p("up_scales"),
                               p("dgate"), p("dup"), p("again"), stream)
        return {n: s[n] for n in ("y", "dgate", "dup", "again")}
    gt.pack_rows(ctx, d, p("x"), p("codes"), p("scales"), stream)
    gt.unpack_rows(ctx, d, p("codes"), p("scales"), p("y"), stream)
    return {"y": s["y"], "scales": s["scales"]}


def _act(z, name):
    """act(z) and its derivative in float32."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, 0.0), (z > 0).float()
    if name == "silu":
        g = 1 / (1 + torch.exp(-z))
        return z * g, g * (1 + z * (1 - g))
    c = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * c, c + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _kept(v, case):
    """(what 8 bits keep of v in float32, the scales)."""
    R, C = v.shape
    B = case["scale_columns"] or C
    blocks = -(-C // B)
    v = torch.cat([v.float(), v.new_zeros(R, blocks * B - C, dtype=torch.float32)], dim=1).view(R, blocks, B)
    most = v.abs().amax(dim=2, keepdim=True)
    scale = (most.double() / (127 if case["codes"] == "int8" else 448)).float()
    if case["codes"] == "int8":
        q = (v.double() / torch.where(scale > 0, scale, 1.0).double())
        q = (torch.sign(q) * torch.floor(q.abs() + 0.5)).clamp(-127, 127).float()
    else:
        q = (v / torch.where(scale > 0, scale, 1.0)).clamp(-448, 448).to(torch.float8_e4m3fn).float()
    return (q * scale).view(R, blocks * B)[:, :C], scale.view(R, blocks)


def _run_plain(s):
    case, t, kind = s["case"], TYPES[s["case"]["values"]], s["case"]["kind"]
    if kind == "route":
        return _route_plain(s)
    if kind == "norm":
        sums = (s["x"].float() + s["residual"].float()).to(t)
        v, w, C = sums.float(), s["w"].float(), case["columns"]
        inverse = 1 / torch.sqrt((v * v).sum(dim=1, keepdim=True) / C + EPSILON)
        y = v * inverse * w
        if case["codes"] != "none":
            y = _kept(y, case)[0]
        out = {"sums": sums, "y": y.to(t)}
        if case["training"]:
            dy, n = s["dy"].float(), v * inverse
            dn = dy * w
            dx = inverse * (dn - n * ((dn * n).sum(dim=1, keepdim=True) / C)) + s["dsum"].float()
            out.update(dx=dx.to(t), dw=(dy * n).sum(dim=0))
        return out
    if kind == "product":
        return _product_plain(s)
    if kind == "activation":
        limit = case["limit"] or math.inf

        def gated(gate, up):
            a, da = _act(torch.clamp(gate, max=limit), case["activation"])
            return a, da * (gate <= limit), torch.clamp(up, -limit, limit), (up.abs() <= limit).float()

        a, _, u, _ = gated(s["gate"].float(), s["up"].float())
        out = {"y": (a * u).to(t)}
        a, da, u, du = gated(_kept(s["gate"], case)[0], _kept(s["up"], case)[0])
        dy = s["dy"].float()
        out.update(dgate=(dy * u * da).to(t), dup=(dy * a * du).to(t), again=(a * u).to(t))
        return out
    kept, scales = _kept(s["x"], case)
    return {"y": kept.to(t), "scales": scales}


def _route_plain(s):
    case = s["case"]
    T, E, k, G = case["tokens"], case["experts"], case["k"], case["groups"]
    l = s["logits"].double()
    if case["scores"] == "softmax":
        e = torch.exp(l - l.amax(dim=1, keepdim=True))
        score = e / e.sum(dim=1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-l))
    # without biases the order is the logits' own
    key = score + s["bias"].double() if case["bias"] else l
    if G > 1:
        of = (key if case["bias"] or case["best"] == 1 else score).view(T, G, E // G)
        sums = torch.sort(of, dim=2, descending=True).values[:, :, :case["best"]].sum(dim=2)
        groups = torch.sort(sums, dim=1, descending=True, stable=True).indices[:, :case["chosen_groups"]]
        inside = torch.zeros(T, G, dtype=torch.bool, device="cuda").scatter_(1, groups, True)
        key = torch.where(inside.repeat_interleave(E // G, dim=1), key, -math.inf)
    chosen = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    mine = score.gather(1, chosen)
    total = mine.sum(dim=1, keepdim=True) if case["renormalize"] else 1.0
    flat = chosen.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    places = torch.empty_like(order)
    places[order] = torch.arange(T * k, device="cuda")
    offsets = torch.searchsorted(flat[order], torch.arange(E + 1, device="cuda"))
    out = {"chosen": chosen.int(), "gates": (case["scale"] * mine / total).float(), "offsets": offsets.int(),
           "rows": (order // k).int(), "places": places.view(T, k).int()}
    if case["training"]:
        dg = s["dgates"].double() * case["scale"]
        ds = torch.zeros_like(l)
        if case["renormalize"]:
            dg = (dg - (dg * mine).sum(dim=1, keepdim=True) / total) / total
        ds.scatter_(1, chosen, dg)
        if case["scores"] == "softmax":
            dl = score * (ds - (ds * score).sum(dim=1, keepdim=True))
        else:
            dl = ds * score * (1 - score)
        out["dlogits"] = dl.to(TYPES[case["values"]])
    return out


def _product_plain(s):
    case, t = s["case"], TYPES[s["case"]["values"]]
    R, G, N = case["rows"], case["groups"], case["outputs"]
    x, w = s["x"].float(), s["w"].float()
    if G > 1:
        # every group's rows padded to the longest's
        offsets, row = s["offsets"].long(), torch.arange(R, device="cuda")
        group = (row[:, None] >= offsets[1:]).sum(dim=1)
        at = group * s["most"] + row - offsets[group]
        padded = x.new_zeros(G * s["most"], case["inputs"])
        padded[at] = x
        z = torch.bmm(padded.view(G, s["most"], -1), w.transpose(1, 2).contiguous()).view(G * s["most"], N)[at]
    else:
        group = torch.zeros(R, dtype=torch.long, device="cuda")
        z = x @ w[0].T
    if case["bias"]:
        z = z + s["b"].float()[group]
    a, _ = _act(z, case["activation"])
    y = a * s["factor"].float() if case["factor"] else a
    if case["residual"]:
        y = y + s["residual"].float()
    out = {"y": y.to(t)}
    if case["training"]:
        z = z.to(t)
        a, da = _act(z.float(), case["activation"])
        dy = s["dy"].float()
        dz = (dy * da * s["factor"].float() if case["factor"] else dy * da).to(t)
        out.update(z=z, dz=dz)
        if case["factor"]:
            out["dfactor"] = (dy * a).to(t)
        if case["bias"]:
            out["db"] = torch.zeros(G, N, device="cuda", dtype=torch.float64).index_add_(0, group, dz.double()).to(t)
    return out


# --------------------------------------------------------------------------
# what one pass cannot do without, and its values in 64 bits
# --------------------------------------------------------------------------

def work(case):
    size, kind = 4 if case["values"] == "f32" else 2, case["kind"]
    if kind == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        n = T * E * size + T * k * 16 + 4 * (E + 1) + (4 * E if case["bias"] else 0)
        if case["training"]:
            n += T * E * size + T * k * 4
        return {"bytes": n, "flops": T * E * (14 if case["training"] else 8)}
    R = case["rows"]
    if kind == "product":
        K, N = case["inputs"], case["outputs"]
        used = int((np.diff(_offsets(case, 0)) > 0).sum())
        rows = K + N * (1 + case["factor"] + case["residual"])
        if case["training"]:  # z and dz, dy, the factor's gradient
            rows += N * (3 + case["factor"])
        n = R * rows * size + used * N * K * size + (used * N * size if case["bias"] else 0)
        if case["training"] and case["bias"]:
            n += case["groups"] * N * size
        return {"bytes": n, "flops": 2 * R * N * K + R * N * (24 if case["training"] else 8)}
    C = case["columns"]
    scales = 0 if case["codes"] == "none" else 4 * R * -(-C // (case["scale_columns"] or C))
    if kind == "norm":
        n = R * C * size * 3 + C * size + (R * C + scales if case["codes"] != "none" else R * C * size)
        if case["codes"] != "none":  # and read back
            n += R * C * size
        if case["training"]:  # dy, the sums' gradients, dx, dw
            n += R * C * size * 3 + 4 * C
        return {"bytes": n, "flops": R * C * (16 if case["training"] else 5)}
    if kind == "activation":  # gate, up, y and what is kept; dy, two gradients and y again
        return {"bytes": R * C * size * 7 + 2 * (R * C + scales), "flops": R * C * 40}
    return {"bytes": 2 * R * C * size + R * C + scales, "flops": R * C * 4}


def _exact_act(z, name):
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.relu(z), (z > 0).double()
    if name == "silu":
        return z * torch.sigmoid(z), torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)
    phi = torch.special.ndtr(z)
    return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def exact(case, seed):
    s, kind, t = _made(case, seed), case["kind"], TYPES[case["values"]]

    def kept_of(v):
        """What 8 bits keep of v, and the float32 scales they go by."""
        v = v.cpu().numpy()
        B = case["scale_columns"] or v.shape[1]
        top = 127.0 if case["codes"] == "int8" else 448.0
        out, scales = np.zeros_like(v), []
        for c in range(0, v.shape[1], B):
            part = v[:, c:c + B]
            scale = (np.abs(part).max(axis=1) / top).astype(np.float32).astype(np.float64)[:, None]
            by = np.where(scale > 0, scale, 1.0)
            if case["codes"] == "int8":
                q = part / by
                q = np.sign(q) * np.floor(np.abs(q) + 0.5)
            else:
                # steps of 2^-3 of the power of two below, 2^-9 at least
                q = (part.astype(np.float32) / by.astype(np.float32)).astype(np.float64)
                step = np.ldexp(1.0, np.maximum(np.frexp(q)[1] - 4, -9))
                q = np.rint(q / step) * step
            out[:, c:c + B] = np.clip(q, -top, top) * scale
            scales.append(scale)
        return torch.from_numpy(out).cuda(), torch.from_numpy(np.concatenate(scales, axis=1)).cuda()

    if kind == "route":
        l = s["logits"].double().cpu().numpy()
        T, E, k, G = case["tokens"], case["experts"], case["k"], case["groups"]
        if case["scores"] == "softmax":
            score = np.exp(l - l.max(axis=1)[:, None])
            score /= score.sum(axis=1)[:, None]
        else:
            score = 1 / (1 + np.exp(-l))
        key = score + s["bias"].double().cpu().numpy() if case["bias"] else l
        of = -np.sort(-(score if not case["bias"] and case["best"] == 2 else key).reshape(T, G, E // G), axis=2)
        best = np.argsort(-of[:, :, :case["best"]].sum(axis=2), axis=1, kind="stable")[:, :case["chosen_groups"]]
        allowed = np.zeros((T, G), bool)
        np.put_along_axis(allowed, best, True, axis=1)
        chosen = np.argsort(np.where(np.repeat(allowed, E // G, axis=1), -key, np.inf), axis=1, kind="stable")[:, :k]
        mine = np.take_along_axis(score, chosen, axis=1)
        total = mine.sum(axis=1)[:, None] if case["renormalize"] else np.ones((T, 1))
        out = {"chosen": None, "gates": torch.from_numpy(case["scale"] * mine / total).cuda(), "offsets": None, "rows": None,
               "places": None}
        if case["training"]:
            # the derivative of gate i by score j, then of the scores by the logits
            dg = s["dgates"].double().cpu().numpy() * case["scale"]
            by_score = dg / total
            if case["renormalize"]:
                by_score = by_score - (dg * mine).sum(axis=1)[:, None] / total ** 2
            if case["scores"] == "softmax":
                dl = -score * (by_score * mine).sum(axis=1)[:, None]
                np.put_along_axis(dl, chosen, np.take_along_axis(dl, chosen, axis=1) + by_score * mine, axis=1)
            else:
                dl = np.zeros_like(l)
                np.put_along_axis(dl, chosen, by_score * mine * (1 - mine), axis=1)
            out["dlogits"] = torch.from_numpy(dl).cuda()
        return out
    if kind == "norm":
        v = s["x"].double() + s["residual"].double()
        out = {"sums": v}
        v = v.to(t).double()  # the norm takes the sums as they are kept
        r, w = torch.rsqrt(v.square().mean(dim=1, keepdim=True) + EPSILON), s["w"].double()
        y = v * r * w
        if case["codes"] != "none":
            y = kept_of(y)[0]
        out["y"] = y
        if case["training"]:
            dy = s["dy"].double()
            dv = dy * w * r - v * r ** 3 * (dy * w * v).mean(dim=1, keepdim=True)
            out.update(dx=dv + s["dsum"].double(), dw=(dy * v * r).sum(dim=0))
        return out
    if kind == "product":
        R, G, N = case["rows"], case["groups"], case["outputs"]
        at = _offsets(case, seed)
        z = torch.zeros(R, N, dtype=torch.float64, device="cuda")
        for g in range(G):
            rows = slice(int(at[g]), int(at[g + 1]))
            z[rows] = torch.mm(s["x"][rows].double(), s["w"][g].double().t())
            if case["bias"]:
                z[rows] += s["b"][g].double()
        a, _ = _exact_act(z, case["activation"])
        y = a * s["factor"].double() if case["factor"] else a
        out = {"y": y + s["residual"].double() if case["residual"] else y}
        if case["training"]:
            out["z"] = z
            # the backward takes z and dz as they are kept
            a, da = _exact_act(z.to(t).double(), case["activation"])
            dz = s["dy"].double() * da * (s["factor"].double() if case["factor"] else 1.0)
            out["dz"] = dz
            if case["factor"]:
                out["dfactor"] = s["dy"].double() * a
            if case["bias"]:
                dz = dz.to(t).double()
                out["db"] = torch.stack([dz[int(at[g]):int(at[g + 1])].sum(dim=0) for g in range(G)])
        return out
    if kind == "activation":
        limit = case["limit"] or math.inf

        def parts(gate, up):
            a, da = _exact_act(gate.clamp(max=limit), case["activation"])
            return a, torch.where(gate > limit, 0.0, da), up.clamp(-limit, limit), torch.where(up.abs() > limit, 0.0, 1.0)

        a, _, u, _ = parts(s["gate"].double(), s["up"].double())
        out = {"y": a * u}
        a, da, u, du = parts(kept_of(s["gate"].double())[0], kept_of(s["up"].double())[0])
        dy = s["dy"].double()
        out.update(dgate=dy * u * da, dup=dy * a * du, again=a * u)
        return out
    kept, scales = kept_of(s["x"].double())
    return {"y": kept, "scales": scales}
