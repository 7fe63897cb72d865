"""The operators of a block in plain rows where rows lie 2^20 values apart and end behind
offsets of 2^32 values: the same bits as with rows close together."""
import pytest
import torch

import gotransformers_amd as gt
from tests.device_rows import say, stream

pytestmark = pytest.mark.gpu

FAR, ROWS = 1 << 20, 4100
BF16 = gt.VALUES_BFLOAT16


@pytest.fixture(scope="module")
def ctx():
    c = gt.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def far():
    """Six buffers of 8 GiB, one of them of bytes, for rows that lie apart."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("80 GiB of device memory are wanted")
    made = [torch.empty(ROWS * FAR, dtype=torch.bfloat16, device="cuda") for _ in range(5)]
    yield made + [torch.empty(ROWS * FAR, dtype=torch.uint8, device="cuda")]
    del made
    torch.cuda.empty_cache()


def apart(buffer, width):
    return buffer.view(ROWS, FAR)[:, :width]


def values(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def same(*pairs):
    torch.cuda.synchronize()
    for a, b in pairs:
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def run_both(far, width, inputs, outputs, call):
    """call(pointers of inputs, of outputs, stride) with rows close together and apart; the
    results of both, in pairs."""
    near = [torch.zeros(ROWS, width, dtype=torch.bfloat16, device="cuda") for _ in range(outputs)]
    views = [apart(b, width) for b in far[:len(inputs) + outputs]]
    for v, x in zip(views, inputs):
        v.copy_(x)
    call([x.data_ptr() for x in inputs], [x.data_ptr() for x in near], width)
    call([v.data_ptr() for v in views[:len(inputs)]], [v.data_ptr() for v in views[len(inputs):]], FAR)
    return list(zip(near, views[len(inputs):]))


@pytest.mark.parametrize("width", [72, 2048])
def test_norm_far_apart(ctx, far, width):
    say("norm", width)
    w, x, r = values(1, width), values(2, ROWS, width), values(3, ROWS, width)

    def forward(i, o, ld):
        d = gt.norm_desc(BF16, ROWS, width, input_stride=ld, residual_stride=ld, sum_stride=ld, output_stride=ld)
        gt.norm_forward(ctx, d, i[0], i[1], w.data_ptr(), o[0], o[1], stream=stream())
    same(*run_both(far, width, [x, r], 2, forward))
    dw = []

    def gradient(i, o, ld):
        d = gt.norm_desc(BF16, ROWS, width, input_stride=ld, sum_stride=ld, output_stride=ld)
        n = gt.norm_workspace_bytes(d)
        ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
        dw.append(torch.zeros(width, device="cuda"))
        gt.norm_gradient(ctx, d, i[0], i[1], w.data_ptr(), i[2], o[0], dw[-1].data_ptr(), gt.VALUES_FLOAT32, False, ws.data_ptr(),
                         stream(), n)
        torch.cuda.synchronize()
    same(*run_both(far, width, [x, r, values(4, ROWS, width)], 1, gradient))
    same(tuple(dw))


def test_packed_rows_and_activations_far_apart(ctx, far):
    say("packed")
    width = 72
    g, u, dy = values(5, ROWS, width), values(6, ROWS, width), values(7, ROWS, width)
    codes, scales = {}, {}

    def pack(i, o, ld):
        codes[ld] = apart(far[5], width) if ld == FAR else torch.zeros(ROWS, width, dtype=torch.uint8, device="cuda")
        scales[ld] = torch.zeros(ROWS, 3, device="cuda")
        d = gt.packed_desc(BF16, ROWS, width, gt.CODES_INT8, 32, value_stride=ld, code_stride=ld)
        gt.pack_rows(ctx, d, i[0], codes[ld].data_ptr(), scales[ld].data_ptr(), stream())
        gt.unpack_rows(ctx, d, codes[ld].data_ptr(), scales[ld].data_ptr(), o[0], stream())
    same(*run_both(far, width, [g], 1, pack))
    same((codes[FAR], codes[width]), (scales[FAR], scales[width]))

    def desc(ld, kept):
        return gt.activation_desc(BF16, ROWS, width, gt.ACTIVATION_SILU, 0.0, kept, 32 if kept else 0, gate_stride=ld, up_stride=ld,
                                  output_stride=ld, code_stride=ld)

    def forward(i, o, ld):
        gt.activation_forward(ctx, desc(ld, 0), i[0], i[1], o[0], stream=stream())
    same(*run_both(far, width, [g, u], 1, forward))

    def gradient(i, o, ld):  # the gates' codes for the ups', which are read alike
        c, s = codes[ld].data_ptr(), scales[ld].data_ptr()
        gt.activation_gradient(ctx, desc(ld, gt.CODES_INT8), i[0], c, s, c, s, o[0], o[1], o[2], stream())
    same(*run_both(far, width, [dy], 3, gradient))


@pytest.mark.parametrize("groups, inputs, width", [(1, 64, 2304), (1, 64, 200), (16, 72, 203)])
def test_fused_products_far_apart(ctx, far, groups, inputs, width):
    say("product", groups, inputs, width)
    offsets = (torch.arange(groups + 1, dtype=torch.int32) * (ROWS // groups)).cuda()
    offsets[-1] = ROWS
    x, w, b = values(8, ROWS, inputs), values(9, groups, width, inputs), values(10, groups, width)

    def call(i, o, ld):
        d = gt.grouped_desc(BF16, groups, ROWS, inputs, width, output_stride=ld)
        e = gt.epilogue(gt.ACTIVATION_SILU, b.data_ptr(), i[0], i[1], o[0], width, factor_stride=ld, residual_stride=ld,
                        product_stride=ld)
        gt.grouped_fused_forward(ctx, d, e, offsets.data_ptr(), x.data_ptr(), w.data_ptr(), o[1], stream())
    pairs = run_both(far, width, [values(11, ROWS, width), values(12, ROWS, width)], 2, call)
    same(*pairs)
    sums = []

    def bias(i, o, ld):
        d = gt.grouped_desc(BF16, groups, ROWS, inputs, width, output_stride=ld)
        n = gt.grouped_bias_workspace_bytes(d)
        ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
        sums.append(torch.zeros(groups, width, device="cuda"))
        gt.grouped_bias_gradient(ctx, d, offsets.data_ptr(), i[0], sums[-1].data_ptr(), gt.VALUES_FLOAT32, False, ws.data_ptr(),
                                 stream(), n)
        torch.cuda.synchronize()
    run_both(far, width, [pairs[0][0]], 0, bias)
    same(tuple(sums))


@pytest.mark.parametrize("experts, k", [(60, 4), (256, 8)])
def test_route_far_apart(ctx, far, experts, k):
    say("route", experts, k)
    logits, dg = values(13, ROWS, experts), torch.randn(ROWS, k, device="cuda")
    found = []

    def call(i, o, ld):
        d = gt.route_desc(BF16, ROWS, experts, k, logit_stride=ld)
        n = gt.route_workspace_bytes(d)
        ws = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda")
        got = [torch.zeros(ROWS, k, dtype=t, device="cuda") for t in (torch.int32, torch.float32, torch.int32, torch.int32)]
        off = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
        gt.route_forward(ctx, d, i[0], None, got[0].data_ptr(), got[1].data_ptr(), off.data_ptr(), got[2].data_ptr(),
                         got[3].data_ptr(), ws.data_ptr(), stream(), n)
        gt.route_gradient(ctx, d, i[0], got[0].data_ptr(), dg.data_ptr(), o[0], stream())
        torch.cuda.synchronize()
        found.append(got + [off])
    same(*run_both(far, experts, [logits], 1, call))
    same(*zip(*found))
