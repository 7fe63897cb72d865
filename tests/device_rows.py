"""Rows inside larger device buffers, for the GPU tests of the operators over plain rows."""
import numpy as np
import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "u8": torch.uint8, "i32": torch.int32}
SENTINEL = 77


def stream():
    return torch.cuda.current_stream().cuda_stream


def say(*a):
    print(*a, flush=True)


class Rows:
    """rows x width values of `kind`, `stride` apart, `shift` values behind the
    start of a buffer that holds SENTINEL everywhere else."""

    def __init__(self, kind, rows, width, stride=None, shift=0, data=None):
        stride = width if stride is None else stride
        n = max(rows, 1) * stride
        self.buffer = torch.full((shift + n + 64,), SENTINEL, dtype=TYPES[kind], device="cuda")
        self.view = self.buffer[shift:shift + n].view(max(rows, 1), stride)[:rows, :width]
        self.kind, self.stride = kind, stride
        if data is not None:
            self.view.copy_(torch.as_tensor(np.ascontiguousarray(data)).to(TYPES[kind]))

    @property
    def ptr(self):
        return self.view.data_ptr()

    def get(self):
        v = self.view
        return (v.double() if v.dtype.is_floating_point else v).cpu().numpy()

    def check_outside(self):
        """Nothing but the rows was written."""
        was = self.view.clone()
        self.view.fill_(SENTINEL)
        assert bool((self.buffer == SENTINEL).all()), "values beside the rows were written"
        self.view.copy_(was)


def rounded(a, kind):
    """float64 values as they are after one rounding to the type."""
    return torch.as_tensor(np.asarray(a)).to(TYPES[kind]).double().numpy()


def strides(width, layout):
    """(stride, shift) of a layout: packed; padded to whole 16 bytes; odd strides and addresses."""
    if layout == "packed":
        return width, 0
    return (-(-width // 16) * 16 + 16, 16) if layout == "padded" else (width + 3, 1)
