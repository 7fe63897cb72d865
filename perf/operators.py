"""Operators over plain rows beside the mixture-of-experts layer, as measurable cases.

  forward, input_gradient, weight_gradient
            the ragged products of experts kept in training precision: rows
            sorted by expert (as gtmoe_last_routing lists them), offsets[e] ..
            offsets[e + 1] the rows of expert e
              y[r] = W_e x[r],  dx[r] = W_e^T dy[r],  dW_e = sum_r dy[r] x[r]^T
  training  the three of them as one projection of a training step
  adapted   a projection that all requests share, beside the low-rank adapter
            of each row's own request (-1: none)
              y[t] = W x[t] + b + s_a B_a A_a x[t]
            or, where the shared product was made elsewhere, added to it
              y[t] + s_a B_a A_a x[t]
  dropout   out = base + keep * x * 65536 / (65536 - t), t = round(65536 rate),
            and the gradient of x by the same call.  keep comes from
            Philox4x32 with ten rounds (Salmon et al., SC 2011): value
            (row, column) takes 16 bits of the words of the counter
            (column / 8, row, offset's low and high half) under the key (seed's
            low and high half) -- the low then the high half of each word in
            turn -- and is kept where they are at least t.

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
GROUPED = ("forward", "input_gradient", "weight_gradient", "training")


def _grouped(kind, shape, T, values, down=False, gradient="same"):
    """down: the projection from h to d instead of from d to h."""
    s = SHAPES[shape]
    K, N = (s["h"], s["d"]) if down else (s["d"], s["h"])
    return dict(kind=kind, values=values, rows=T * s["k"], groups=s["E"], inputs=K, outputs=N, zipf=s["zipf"],
                gradient=gradient)


def _adapted(T, inputs, outputs, rank, adapters, run, values, none=0.0, shared=True):
    """run: consecutive rows of one request; none: share of requests without an adapter."""
    return dict(kind="adapted", values=values, rows=T, inputs=inputs, outputs=outputs, rank=rank, adapters=adapters,
                run=run, none=none, shared=shared)


def _dropout(rows, columns, rate, values, residual):
    return dict(kind="dropout", values=values, rows=rows, columns=columns, rate=rate, residual=residual)


def listed():
    cases = {
        # a decode batch of 32 sequences through 16 experts: four rows each, the weights' bytes
        "forward_bf16_decode": _grouped("forward", "wide", 32, "bf16"),
        # a prompt of 4096 tokens over many small experts
        "forward_bf16_prefill": _grouped("forward", "many", 4096, "bf16"),
        # full precision with ragged widths, as a numerics check or a small model trains
        "training_f32_ragged": _grouped("training", "ragged", 777, "f32", gradient="f32"),
        # what the experts hand back to the layer below
        "input_gradient_bf16": _grouped("input_gradient", "wide", 8192, "bf16"),
        # what the optimizer takes, summed in full precision
        "weight_gradient_bf16": _grouped("weight_gradient", "block", 4096, "bf16", down=True, gradient="f32"),
        # one projection of a long, skewed training batch
        "training_f16_skewed": _grouped("training", "skewed", 16384, "f16"),
        # one generated token of one request
        "adapted_bf16_t1": _adapted(1, 2048, 2048, 16, 8, 1, "bf16"),
        # a decode batch whose requests each bring their own adapter, a few none
        "adapted_bf16_t64": _adapted(64, 2048, 2048, 16, 48, 1, "bf16", none=0.2),
        # prompts of several requests packed into one batch
        "adapted_f16_prefill": _adapted(8192, 1024, 2048, 64, 12, 700, "f16", none=0.1),
        # ragged widths, added to a shared product made elsewhere
        "adapted_f32_ragged": _adapted(333, 1000, 1201, 8, 5, 37, "f32", none=0.2, shared=False),
        # a residual branch of a training batch
        "dropout_bf16": _dropout(8192, 2048, 0.1, "bf16", True),
        # an adapter's input, odd widths
        "dropout_f32_ragged": _dropout(2331, 1201, 0.25, "f32", False),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["forward", "forward", "input_gradient", "weight_gradient", "training", "adapted", "adapted",
                       "adapted", "dropout"])
    values = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in GROUPED:
        shape = rng.choice(list(SHAPES))
        top = 2048 if values == "f32" else 8192
        T = log_int(1 if kind in ("forward", "input_gradient") else 8, top)
        return _grouped(kind, shape, T, values, down=rng.random() < 0.4, gradient=rng.choice(["same", "f32"]))
    if kind == "adapted":
        shape = SHAPES[rng.choice(list(SHAPES))]
        sides = [shape["d"], shape["h"]]
        rng.shuffle(sides)
        T = log_int(1, 2048 if values == "f32" else 8192)
        run = 1 if T <= 256 and rng.random() < 0.6 else log_int(2, max(2, T))
        adapters = log_int(1, min(64, max(1, -(-T // run))))
        return _adapted(T, sides[0], sides[1], rng.choice([4, 8, 16, 24, 32, 64]), adapters, run, values,
                        none=rng.choice([0.0, 0.0, 0.3]), shared=rng.random() < 0.75)
    return _dropout(log_int(1, 8192), log_int(8, 2048), round(rng.uniform(0.05, 0.6), 3), values, rng.random() < 0.5)


# --------------------------------------------------------------------------
# inputs, from the seed alone
# --------------------------------------------------------------------------

def _plan(case, seed):
    """The whole numbers of the case: the experts' offsets or the rows' adapters."""
    g = np.random.default_rng([seed, case["rows"], 77])
    if case["kind"] in GROUPED:
        E = case["groups"]
        p = 1.0 / np.arange(1, E + 1) ** case["zipf"]
        sizes = g.multinomial(case["rows"], g.permutation(p / p.sum()))
        return np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    requests = -(-case["rows"] // case["run"])
    chosen = np.concatenate([g.permutation(case["adapters"])[:requests],
                             g.integers(0, case["adapters"], max(0, requests - case["adapters"]))])
    chosen = np.where(g.random(requests) < case["none"], -1, g.permutation(chosen))
    return np.repeat(chosen, case["run"])[:case["rows"]].astype(np.int32)


def _made(case, seed):
    """The arrays of the case on the GPU."""
    t = TYPES[case["values"]]
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + case["rows"])

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype or t)

    if case["kind"] == "dropout":
        r, c = case["rows"], case["columns"]
        return dict(x=normal(r, c), dy=normal(r, c), base=normal(r, c) if case["residual"] else None,
                    seed=int(seed) * 1000003 + 17, offset=int(seed) + (1 << 32))
    R, K, N = case["rows"], case["inputs"], case["outputs"]
    if case["kind"] in GROUPED:
        E = case["groups"]
        offsets = _plan(case, seed)
        m = dict(offsets=torch.from_numpy(offsets).cuda(), bounds=offsets.tolist())
        m["x"] = normal(R, K)
        m["w"] = normal(E, N, K, scale=K ** -0.5)
        m["dy"] = normal(R, N)
        return m
    n, r = case["adapters"], case["rank"]
    m = dict(adapter=torch.from_numpy(_plan(case, seed)).cuda(), x=normal(R, K))
    m["w"] = normal(N, K, scale=K ** -0.5) if case["shared"] else None
    m["b"] = normal(N, scale=0.1) if case["shared"] else None
    m["base"] = None if case["shared"] else normal(R, N)
    m["down"], m["up"] = normal(n, r, K, scale=K ** -0.5), normal(n, N, r, scale=r ** -0.5)
    m["scales"] = torch.rand(n, generator=g, device="cuda") + 0.5
    return m


_context = None


def prepare(case, seed):
    s = _made(case, seed)
    s["case"] = case
    if not own:
        return s
    import gotransformers_amd as gt

    global _context
    if _context is None:
        _context = gt.Context(0)
    t = TYPES[case["values"]]
    values = {"f32": gt.VALUES_FLOAT32, "bf16": gt.VALUES_BFLOAT16, "f16": gt.VALUES_FLOAT16}

    def empty(*shape, dtype=t):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    if case["kind"] == "dropout":
        s["desc"] = gt.dropout_desc(values[case["values"]], case["rows"], case["columns"])
        s["y"], s["dx"] = empty(case["rows"], case["columns"]), empty(case["rows"], case["columns"])
        return s
    R, K, N = case["rows"], case["inputs"], case["outputs"]
    if case["kind"] in GROUPED:
        s["desc"] = gt.grouped_desc(values[case["values"]], case["groups"], R, K, N)
        s["y"], s["dx"] = empty(R, N), empty(R, K)
        s["gradient"] = values["f32"] if case["gradient"] == "f32" else values[case["values"]]
        s["dw"] = empty(case["groups"], N, K, dtype=torch.float32 if case["gradient"] == "f32" else t)
        return s
    s["desc"] = gt.adapted_desc(values[case["values"]], R, K, N, case["adapters"], case["rank"])
    s["workspace"] = empty(gt.adapted_workspace_bytes(s["desc"]), dtype=torch.uint8)
    s["y"] = empty(R, N)
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import gotransformers_amd as gt

    case, ctx = s["case"], _context
    stream = torch.cuda.current_stream().cuda_stream

    def p(t):
        return None if t is None else t.data_ptr()

    kind = case["kind"]
    if kind == "dropout":
        gt.dropout(ctx, s["desc"], p(s["x"]), p(s["base"]), p(s["y"]), case["rate"], s["seed"], s["offset"], stream)
        gt.dropout(ctx, s["desc"], p(s["dy"]), None, p(s["dx"]), case["rate"], s["seed"], s["offset"], stream)
        return s["y"], s["dx"]
    if kind == "adapted":
        if not case["shared"]:
            s["y"].copy_(s["base"])
        gt.adapted_forward(ctx, s["desc"], p(s["x"]), p(s["w"]), p(s["b"]), p(s["adapter"]), p(s["down"]), p(s["up"]),
                           p(s["scales"]), p(s["y"]), p(s["workspace"]), stream)
        return s["y"]
    out = []
    if kind in ("forward", "training"):
        gt.grouped_forward(ctx, s["desc"], p(s["offsets"]), p(s["x"]), p(s["w"]), p(s["y"]), stream)
        out.append(s["y"])
    if kind in ("input_gradient", "training"):
        gt.grouped_input_gradient(ctx, s["desc"], p(s["offsets"]), p(s["dy"]), p(s["w"]), p(s["dx"]), stream)
        out.append(s["dx"])
    if kind in ("weight_gradient", "training"):
        gt.grouped_weight_gradient(ctx, s["desc"], p(s["offsets"]), p(s["dy"]), p(s["x"]), p(s["dw"]), s["gradient"],
                                   False, stream)
        out.append(s["dw"])
    return tuple(out)


def _keep(case, seed, offset):
    """The kept places of a rows x columns mask, by Philox4x32-10 in 64-bit integers."""
    low = 0xFFFFFFFF
    blocks = -(-case["columns"] // 8)
    column = torch.arange(blocks, device="cuda", dtype=torch.int64)
    row = torch.arange(case["rows"], device="cuda", dtype=torch.int64)
    c0 = column[None, :].expand(case["rows"], blocks)
    c1 = row[:, None].expand(case["rows"], blocks)
    c2 = torch.full_like(c0, offset & low)
    c3 = torch.full_like(c0, (offset >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low

    def product(a, m):  # high and low 32 bits of a 32 x 32 product, without leaving 63 bits
        upper, lower = (a >> 16) * m, (a & 0xFFFF) * m
        s = upper + (lower >> 16)
        return s >> 16, ((s & 0xFFFF) << 16) | (lower & 0xFFFF)

    for _ in range(10):
        h0, l0 = product(c0, 0xD2511F53)
        h1, l1 = product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    halves = [v for c in (c0, c1, c2, c3) for v in (c & 0xFFFF, c >> 16)]
    bits = torch.stack(halves, dim=2).reshape(case["rows"], 8 * blocks)[:, :case["columns"]]
    return bits >= _threshold(case)


def _threshold(case):
    return int(math.floor(case["rate"] * 65536 + 0.5))


def _run_plain(s):
    case, kind, t = s["case"], s["case"]["kind"], TYPES[s["case"]["values"]]
    if kind == "dropout":
        keep = _keep(case, s["seed"], s["offset"])
        scale = 65536.0 / (65536 - _threshold(case))
        y = torch.where(keep, s["x"].float() * scale, 0.0)
        if case["residual"]:
            y = s["base"].float() + y
        return y.to(t), torch.where(keep, s["dy"].float() * scale, 0.0).to(t)
    if kind == "adapted":
        x, a = s["x"].float(), s["adapter"]
        y = x @ s["w"].float().T + s["b"].float() if case["shared"] else s["base"].float()
        for i in range(case["adapters"]):
            u = (x @ s["down"][i].float().T) * s["scales"][i]
            y = torch.where((a == i)[:, None], y + u @ s["up"][i].float().T, y)
        return y.to(t)
    at = s["bounds"]
    spans = [(e, at[e], at[e + 1]) for e in range(case["groups"])]
    out = []
    if kind in ("forward", "training"):
        out.append(torch.cat([s["x"][i:j].float() @ s["w"][e].float().T for e, i, j in spans]).to(t))
    if kind in ("input_gradient", "training"):
        out.append(torch.cat([s["dy"][i:j].float() @ s["w"][e].float() for e, i, j in spans]).to(t))
    if kind in ("weight_gradient", "training"):
        dw = torch.stack([s["dy"][i:j].float().T @ s["x"][i:j].float() for _, i, j in spans])
        out.append(dw if case["gradient"] == "f32" else dw.to(t))
    return tuple(out)


# --------------------------------------------------------------------------
# what one pass cannot do without, and its values in 64 bits
# --------------------------------------------------------------------------

def work(case):
    size = 4 if case["values"] == "f32" else 2
    kind = case["kind"]
    if kind == "dropout":
        n = case["rows"] * case["columns"]
        return {"bytes": n * size * (5 if case["residual"] else 4), "flops": n * (5 if case["residual"] else 4)}
    R, K, N = case["rows"], case["inputs"], case["outputs"]
    if kind == "adapted":
        a = _plan(case, 0)
        used, rows, r = len(set(a[a >= 0].tolist())), int((a >= 0).sum()), case["rank"]
        values = R * (K + N) + used * r * (K + N) + (N * K + N if case["shared"] else R * N)
        return {"bytes": values * size + 4 * R + 4 * used,
                "flops": (2 * R * N * K if case["shared"] else 0) + 2 * rows * r * (K + N)}
    E = case["groups"]
    weights = int((np.diff(_plan(case, 0)) > 0).sum()) * N * K * size
    dw = E * N * K * (4 if case["gradient"] == "f32" else size)
    parts = {"forward": R * (K + N) * size + weights, "input_gradient": R * (K + N) * size + weights,
             "weight_gradient": R * (K + N) * size + dw}
    if kind == "training":  # x, dy and the weights once, y, dx and dw once
        return {"bytes": 2 * R * (K + N) * size + weights + dw + 4 * (E + 1), "flops": 6 * R * K * N}
    return {"bytes": parts[kind] + 4 * (E + 1), "flops": 2 * R * K * N}


def exact(case, seed):
    s = _made(case, seed)
    kind = case["kind"]
    if kind == "dropout":
        mask = np.uint64(0xFFFFFFFF)
        cols, rows = case["columns"], case["rows"]
        blocks = (cols + 7) // 8
        c = [np.tile(np.arange(blocks, dtype=np.uint64), rows), np.repeat(np.arange(rows, dtype=np.uint64), blocks),
             np.full(rows * blocks, s["offset"] % 2 ** 32, np.uint64),
             np.full(rows * blocks, s["offset"] // 2 ** 32, np.uint64)]
        key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32 % 2 ** 32]
        for i in range(10):
            ki = [np.uint64((key[0] + i * 0x9E3779B9) % 2 ** 32), np.uint64((key[1] + i * 0xBB67AE85) % 2 ** 32)]
            p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(p1 >> np.uint64(32)) ^ c[1] ^ ki[0], p1 & mask, (p0 >> np.uint64(32)) ^ c[3] ^ ki[1], p0 & mask]
        words = np.stack(c, axis=1).astype(np.uint32).view(np.uint16).reshape(rows, 8 * blocks)[:, :cols]
        t = round(case["rate"] * 65536)
        factor = torch.from_numpy((words.astype(np.int64) >= t) * (65536.0 / (65536 - t))).cuda()
        y = s["x"].double() * factor
        return (y + s["base"].double() if case["residual"] else y), s["dy"].double() * factor
    if kind == "adapted":
        x, a = s["x"].double(), s["adapter"].long()
        y = s["base"].double() if not case["shared"] else torch.addmm(s["b"].double(), x, s["w"].double().t())
        for i in sorted(set(a.tolist()) - {-1}):
            at = torch.nonzero(a == i)[:, 0]
            delta = s["up"][i].double() @ (s["down"][i].double() @ x[at].t())
            y[at] += s["scales"][i].double() * delta.t()
        return y
    R, K, N, E = case["rows"], case["inputs"], case["outputs"], case["groups"]
    y = torch.zeros(R, N, dtype=torch.float64, device="cuda")
    dx = torch.zeros(R, K, dtype=torch.float64, device="cuda")
    dw = torch.zeros(E, N, K, dtype=torch.float64, device="cuda")
    for e in range(E):
        rows = slice(s["bounds"][e], s["bounds"][e + 1])
        x, dy, w = s["x"][rows].double(), s["dy"][rows].double(), s["w"][e].double()
        y[rows], dx[rows], dw[e] = torch.mm(x, w.t()), torch.mm(dy, w), torch.mm(dy.t(), x)
    return {"forward": (y,), "input_gradient": (dx,), "weight_gradient": (dw,), "training": (y, dx, dw)}[kind]
