"""The operators of a block in plain rows as a program uses them together: one
training step of x + MoE(norm(x)) whose experts are kept in training precision,
eagerly, captured into a graph, on two streams; and the errors every call shares.

The step's 64-bit form (`reference`) is checked against autograd where nothing
is kept in 8 bits.  Bounds: every stage is off by at most (K + 16) 2^-24, about 2^-17
here, of its terms' sizes; the gradients pass about ten stages, cancellation in a
row's sums allowed a factor of eight: 2^-11 of each result's largest value."""
import numpy as np
import pytest
import torch

import gotransformers_amd as gt
from tests import plain_block as plain
from tests.device_rows import TYPES, say, stream
from tests.plain_rows import VALUES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = gt.Context(0)
    yield c
    c.close()


class Step:
    """Buffers and one step: T tokens of d values, E experts of h, k per token."""

    def __init__(self, kind, T, d, h, E, k, codes, seed, scores=gt.SCORES_SOFTMAX):
        self.kind, self.T, self.d, self.h, self.E, self.k, self.codes = kind, T, d, h, E, k, codes
        g = torch.Generator().manual_seed(seed)
        t = TYPES[kind]
        make = lambda *s, f=1.0: (torch.randn(*s, generator=g, dtype=torch.float64) * f).to(t).cuda()
        self.x, self.r, self.dy = make(T, d), make(T, d), make(T, d)
        self.p = dict(wn=make(d, f=0.1), wr=make(E, d, f=d ** -0.5), br=make(E, f=0.3), wg=make(E, h, d, f=d ** -0.5),
                      bg=make(E, h, f=0.3), wu=make(E, h, d, f=d ** -0.5), wd=make(E, d, h, f=h ** -0.5), bd=make(E, d, f=0.3))
        self.p["wn"] += 1
        self.balance = (torch.randn(E, generator=g) * 0.01).cuda()
        P = T * k
        e = lambda *s, dtype=t: torch.zeros(*s, dtype=dtype, device="cuda")
        self.b = dict(s=e(T, d), y=e(T, d), logits=e(T, E), xs=e(P, d), gz=e(P, h), u=e(P, h), hid=e(P, h), o=e(P, d), do=e(P, d),
                      dh=e(P, h), dg=e(P, h), du=e(P, h), again=e(P, h), dxs=e(P, d), dxs2=e(P, d), dlogits=e(T, E), dyr=e(T, d),
                      dyn=e(T, d), dx=e(T, d))
        self.i = {n: e(*s, dtype=torch.int32) for n, s in dict(chosen=(T, k), off=(E + 1,), rows=(P,), places=(T, k)).items()}
        self.f = {n: e(*s, dtype=torch.float32) for n, s in dict(gates=(T, k), dgates=(T, k), dwn=(d,), dwr=(E, d), dbr=(E,), dwg=(E, h, d),
                                                                dbg=(E, h), dwu=(E, h, d), dwd=(E, d, h), dbd=(E, d)).items()}
        V = VALUES[kind]
        self.norm = gt.norm_desc(V, T, d)
        self.route = gt.route_desc(V, T, E, k, scores=scores, scale=1.5)
        self.router, self.up, self.down = gt.grouped_desc(V, 1, T, d, E), gt.grouped_desc(V, E, P, d, h), gt.grouped_desc(V, E, P, h, d)
        self.act = gt.activation_desc(V, P, h, gt.ACTIVATION_SILU, 4.0, codes, 32 if codes else 0)
        blocks = -(-h // 32)
        self.kept = [(e(P, h, dtype=torch.uint8), e(P, blocks, dtype=torch.float32)) for _ in range(2)]
        sizes = [gt.norm_workspace_bytes(self.norm), gt.route_workspace_bytes(self.route)]
        sizes += [gt.grouped_bias_workspace_bytes(x) for x in (self.router, self.up, self.down)]
        self.ws = e(max(sizes), dtype=torch.uint8)

    def run(self, ctx):
        b, i, f, s = self.b, self.i, self.f, stream()
        q = {n: t.data_ptr() for part in (self.p, b, i, f) for n, t in part.items()}
        ws, F32, off = self.ws.data_ptr(), gt.VALUES_FLOAT32, q["off"]
        # forward
        gt.norm_forward(ctx, self.norm, self.x.data_ptr(), self.r.data_ptr(), q["wn"], q["s"], q["y"], None, None, s)
        gt.grouped_fused_forward(ctx, self.router, gt.epilogue(biases_ptr=q["br"], width=self.E), None, q["y"], q["wr"], q["logits"], s)
        gt.route_forward(ctx, self.route, q["logits"], self.balance.data_ptr(), q["chosen"], q["gates"], off, q["rows"], q["places"], ws, s)
        torch.index_select(b["y"], 0, i["rows"], out=b["xs"])
        gt.grouped_fused_forward(ctx, self.up, gt.epilogue(biases_ptr=q["bg"], width=self.h), off, q["xs"], q["wg"], q["gz"], s)
        gt.grouped_forward(ctx, self.up, off, q["xs"], q["wu"], q["u"], s)
        kept = [t.data_ptr() for pair in self.kept for t in pair] if self.codes else [None] * 4
        gt.activation_forward(ctx, self.act, q["gz"], q["u"], q["hid"], *kept, s)
        gt.grouped_fused_forward(ctx, self.down, gt.epilogue(biases_ptr=q["bd"], width=self.d), off, q["hid"], q["wd"], q["o"], s)
        at = i["places"].long().reshape(-1)
        mine = b["o"][at].view(self.T, self.k, self.d).float()
        out = (b["s"].float() + (mine * f["gates"][:, :, None]).sum(dim=1)).to(b["o"].dtype)
        # backward
        dy = self.dy.float()
        f["dgates"].copy_((mine * dy[:, None]).sum(dim=2))
        b["do"].index_copy_(0, at, (dy[:, None] * f["gates"][:, :, None]).reshape(-1, self.d).to(b["do"].dtype))
        gt.grouped_input_gradient(ctx, self.down, off, q["do"], q["wd"], q["dh"], s)
        saved = kept if self.codes else [q["gz"], None, q["u"], None]
        gt.activation_gradient(ctx, self.act, q["dh"], *saved, q["dg"], q["du"], q["again"], s)
        gt.grouped_weight_gradient(ctx, self.down, off, q["do"], q["again"], q["dwd"], F32, False, s)
        gt.grouped_bias_gradient(ctx, self.down, off, q["do"], q["dbd"], F32, False, ws, s)
        gt.grouped_weight_gradient(ctx, self.up, off, q["dg"], q["xs"], q["dwg"], F32, False, s)
        gt.grouped_bias_gradient(ctx, self.up, off, q["dg"], q["dbg"], F32, False, ws, s)
        gt.grouped_weight_gradient(ctx, self.up, off, q["du"], q["xs"], q["dwu"], F32, False, s)
        gt.grouped_input_gradient(ctx, self.up, off, q["dg"], q["wg"], q["dxs"], s)
        gt.grouped_input_gradient(ctx, self.up, off, q["du"], q["wu"], q["dxs2"], s)
        gt.route_gradient(ctx, self.route, q["logits"], q["chosen"], q["dgates"], q["dlogits"], s)
        both = (b["dxs"].float() + b["dxs2"].float())[at].view(self.T, self.k, self.d).sum(dim=1)
        gt.grouped_input_gradient(ctx, self.router, self.whole.data_ptr(), q["dlogits"], q["wr"], q["dyr"], s)
        gt.grouped_weight_gradient(ctx, self.router, self.whole.data_ptr(), q["dlogits"], q["y"], q["dwr"], F32, False, s)
        gt.grouped_bias_gradient(ctx, self.router, None, q["dlogits"], q["dbr"], F32, False, ws, s)
        b["dyn"].copy_(both + b["dyr"].float())
        gt.norm_gradient(ctx, self.norm, q["dyn"], q["s"], q["wn"], self.dy.data_ptr(), q["dx"], q["dwn"], F32, False, ws, s)
        return dict(out=out, dx=b["dx"], gates=f["gates"], chosen=i["chosen"], **{n: f[n] for n in f if n.startswith("dw") or n.startswith("db")})

    @property
    def whole(self):
        if not hasattr(self, "_whole"):
            self._whole = torch.tensor([0, self.T], dtype=torch.int32, device="cuda")
        return self._whole

    def reference(self, chosen):
        """The step in 64 bits on the CPU with the device's choice of experts; autograd's
        gradients, but where gate and up are kept in 8 bits the backward reads those."""
        kept = None
        if self.codes:
            name = {gt.CODES_INT8: "int8", gt.CODES_E4M3: "e4m3"}[self.codes]

            class Kept(torch.autograd.Function):
                @staticmethod
                def forward(c, g, u):
                    back = lambda v: torch.from_numpy(plain.unpacked(*plain.packed(v.detach().float().numpy(), name, 32), 32))
                    c.save_for_backward(back(g), back(u))
                    return torch.nn.functional.silu(g.clamp(max=4.0)) * u.clamp(-4.0, 4.0)

                @staticmethod
                def backward(c, dh):
                    g, u = c.saved_tensors
                    with torch.enable_grad():
                        g, u = g.requires_grad_(), u.requires_grad_()
                        y = torch.nn.functional.silu(g.clamp(max=4.0)) * u.clamp(-4.0, 4.0)
                        return torch.autograd.grad(y, (g, u), dh)

            kept = Kept.apply
        p = {n: t.double().cpu().requires_grad_() for n, t in self.p.items()}
        s = (self.x.double() + self.r.double()).cpu().requires_grad_()
        y = s * torch.rsqrt(s.square().mean(dim=1, keepdim=True) + 1e-6) * p["wn"]
        logits = y @ p["wr"].T + p["br"]
        score = torch.softmax(logits, dim=1) if self.route.scores == gt.SCORES_SOFTMAX else torch.sigmoid(logits)
        mine = score.gather(1, chosen.cpu().long())
        gates = 1.5 * mine / mine.sum(dim=1, keepdim=True)
        out = s.clone()
        for e in range(self.E):
            t, j = torch.nonzero(chosen.cpu() == e, as_tuple=True)
            g, u = y[t] @ p["wg"][e].T + p["bg"][e], y[t] @ p["wu"][e].T
            hid = kept(g, u) if kept else torch.nn.functional.silu(g.clamp(max=4.0)) * u.clamp(-4.0, 4.0)
            out = out.index_add(0, t, gates[t, j][:, None] * (hid @ p["wd"][e].T + p["bd"][e]))
        (out * self.dy.double().cpu()).sum().backward()
        want = dict(out=out.detach(), dx=s.grad, gates=gates.detach())
        want.update({"d" + n: t.grad for n, t in p.items()})
        return want


@pytest.mark.parametrize("T, d, h, E, k", [(70, 64, 96, 8, 2), (300, 100, 72, 14, 3)])
@pytest.mark.parametrize("scores", [gt.SCORES_SOFTMAX, gt.SCORES_SIGMOID])
def test_training_step_against_autograd(ctx, T, d, h, E, k, scores):
    step = Step("f32", T, d, h, E, k, gt.CODES_NONE, 1, scores)
    got = step.run(ctx)
    want = step.reference(got["chosen"])
    for n, w in want.items():
        off = (got[n].double().cpu() - w).abs().max() / w.abs().max()
        say(n, float(off))
        assert off <= 2.0 ** -11, n


@pytest.mark.parametrize("codes", [gt.CODES_INT8, gt.CODES_E4M3])
def test_training_step_from_8_bit_checkpoints(ctx, codes):
    """All gradients but the down matrices' (whose inputs are made again from what was kept) follow
    from the kept values; a value next to the border of two codes may be kept one code
    further, so that single gradients move: compared in the 2-norm, to 2^-7."""
    step = Step("f32", 150, 64, 96, 8, 2, codes, 2)
    got = step.run(ctx)
    want = step.reference(got["chosen"])
    for n, w in want.items():
        off = (got[n].double().cpu() - w).norm() / w.norm()
        say(n, float(off))
        # the down matrices see y made again: half a step of 127 or 2^-4 of each value of gate and up
        assert off <= (2.0 ** -11 if n in ("out", "gates") else 2.0 ** -3 if n == "dwd" else 2.0 ** -7), n


@pytest.mark.parametrize("kind, codes, T", [("bf16", gt.CODES_INT8, 300), ("f16", gt.CODES_NONE, 40), ("f32", gt.CODES_E4M3, 700)])
def test_training_step_captured(ctx, kind, codes, T):
    """Replayed after other inputs, with the program's own eager work between: the eager step's bits."""
    step = Step(kind, T, 64, 96, 8, 2, codes, 3)
    other = Step(kind, T, 64, 96, 8, 2, codes, 4)
    step.whole, other.whole
    first = {n: t.clone() for n, t in step.run(ctx).items()}
    second = {n: t.clone() for n, t in other.run(ctx).items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step.run(ctx)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            out = step.run(ctx)
    x, r, dy = step.x.clone(), step.r.clone(), step.dy.clone()
    p = {n: t.clone() for n, t in step.p.items()}
    balance = step.balance.clone()
    for i in range(4):
        for t in out.values():
            t.zero_() if not t.dtype.is_floating_point else t.fill_(float("nan"))
        want, src = (first, None) if i % 2 == 0 else (second, other)
        step.x.copy_(src.x if src else x)
        step.r.copy_(src.r if src else r)
        step.dy.copy_(src.dy if src else dy)
        step.balance.copy_(src.balance if src else balance)
        for n in step.p:
            step.p[n].copy_(src.p[n] if src else p[n])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for n, w in want.items():
            assert torch.equal(out[n], w), (i, n)
        other.run(ctx)  # eager work beside it
        torch.cuda.synchronize()


def test_training_steps_on_two_streams(ctx):
    steps = [Step("bf16", 500, 128, 96, 8, 2, gt.CODES_INT8, 5 + i) for i in range(2)]
    want = []
    for s in steps:
        s.whole
        want.append({n: t.clone() for n, t in s.run(ctx).items()})
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(3):
        got = []
        for s, q in zip(steps, streams):
            with torch.cuda.stream(q):
                got.append(s.run(ctx))
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            for n in w:
                assert torch.equal(g[n], w[n]), n


def test_route_lists_agree_with_the_grouped_products(ctx):
    """What route_forward lists is what the grouped products take: every token's choice j
    lies at places[t][j], in its expert's rows."""
    T, E, k = 777, 14, 3
    l = torch.randn(T, E, device="cuda")
    d = gt.route_desc(gt.VALUES_FLOAT32, T, E, k)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    chosen, gates, off, rows, places = i32(T, k), torch.zeros(T, k, device="cuda"), i32(E + 1), i32(T * k), i32(T, k)
    ws = torch.zeros(gt.route_workspace_bytes(d), dtype=torch.uint8, device="cuda")
    gt.route_forward(ctx, d, l.data_ptr(), None, chosen.data_ptr(), gates.data_ptr(), off.data_ptr(), rows.data_ptr(), places.data_ptr(),
                     ws.data_ptr(), stream())
    eye = torch.arange(1, E + 1, device="cuda", dtype=torch.float32).view(E, 1, 1).contiguous()  # expert e multiplies by e + 1
    x = (torch.arange(T, device="cuda", dtype=torch.float32) + 1)[rows.long()].view(-1, 1).contiguous()
    y = torch.zeros(T * k, 1, device="cuda")
    gt.grouped_forward(ctx, gt.grouped_desc(gt.VALUES_FLOAT32, E, T * k, 1, 1), off.data_ptr(), x.data_ptr(), eye.data_ptr(), y.data_ptr(),
                       stream())
    got = y[places.long().reshape(-1), 0].view(T, k)
    assert torch.equal(got, (torch.arange(T, device="cuda")[:, None] + 1.0) * (chosen + 1))


CALLS = {
    "gtmoe_pack_rows": lambda c, p: gt.pack_rows(c, gt.packed_desc(0, 1, 8, gt.CODES_INT8, 16), p, p + 256, p + 512, stream()),
    "gtmoe_unpack_rows": lambda c, p: gt.unpack_rows(c, gt.packed_desc(0, 1, 8, gt.CODES_INT8, 16), p, p + 256, p + 512, stream()),
    "gtmoe_norm_forward": lambda c, p: gt.norm_forward(c, gt.norm_desc(0, 1, 8), p, None, None, None, p + 256, stream=stream()),
    "gtmoe_norm_gradient": lambda c, p: gt.norm_gradient(c, gt.norm_desc(0, 1, 8), p, p + 256, None, None, p + 512, None, 0, stream=stream()),
    "gtmoe_activation_forward": lambda c, p: gt.activation_forward(c, gt.activation_desc(0, 1, 8, 2), p, None, p + 256, stream=stream()),
    "gtmoe_activation_gradient": lambda c, p: gt.activation_gradient(c, gt.activation_desc(0, 1, 8, 2), p, p + 256, None, None, None, p + 512,
                                                                     None, stream=stream()),
    "gtmoe_grouped_fused_forward": lambda c, p: gt.grouped_fused_forward(c, gt.grouped_desc(0, 1, 1, 8, 8), gt.epilogue(), None, p, p + 256,
                                                                         p + 1024, stream()),
    "gtmoe_grouped_bias_gradient": lambda c, p: gt.grouped_bias_gradient(c, gt.grouped_desc(0, 1, 1, 8, 8), None, p, p + 256, 0, False,
                                                                         p + 1024, stream()),
    "gtmoe_route_forward": lambda c, p: gt.route_forward(c, gt.route_desc(0, 1, 8, 2), p, None, p + 256, p + 512, stream=stream()),
    "gtmoe_route_gradient": lambda c, p: gt.route_gradient(c, gt.route_desc(0, 1, 8, 2), p, p + 256, p + 512, p + 1024, stream()),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_errors_every_call_shares(ctx, name):
    buffer = torch.zeros(65536, dtype=torch.uint8, device="cuda")
    gt.inject_failure(name, gt.ERR_DEVICE)
    with pytest.raises(gt.GtmoeError, match=f"injected failure in {name}"):
        CALLS[name](ctx, buffer.data_ptr())
    ctx.timing_reset()
    ctx.timing(True)
    CALLS[name](ctx, buffer.data_ptr())
    times = ctx.timing_read()
    ctx.timing(False)
    ctx.timing_reset()
    assert times[name[len("gtmoe_"):]][1] == 1
    closed = gt.Context(0)
    gt.library().gtmoe_close(closed.handle)
    with pytest.raises(gt.InvalidArgument, match="context is closed"):
        CALLS[name](closed, buffer.data_ptr())
    closed.close()


def test_nothing_is_allocated(ctx):
    step = Step("bf16", 100, 64, 96, 8, 2, gt.CODES_INT8, 9)
    step.run(ctx)
    before = gt.device_allocations()
    step.run(ctx)
    torch.cuda.synchronize()
    assert gt.device_allocations() == before
