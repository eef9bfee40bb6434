"""Matrices with guards, for the tests of the operators around a layer's products."""
import torch

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# A rounding is off by half a step at most.
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
MARK = 0x5A


class Matrix:
    """Rows (the library's columns) of `cols` values, `ld` apart, `shift` values
    after an address of 256 bytes, all else filled with a mark."""

    def __init__(self, rows, cols, dtype, ld=None, shift=0, data=None):
        self.rows, self.cols, self.ld, self.shift = rows, cols, cols if ld is None else ld, shift
        size = torch.empty(0, dtype=dtype).element_size()
        self.bytes = torch.full(((shift + rows * self.ld + 64) * size,), MARK, dtype=torch.uint8,
                                device="cuda")
        self.flat = self.bytes.view(dtype)
        self.view = self.flat[shift:shift + rows * self.ld].view(rows, self.ld)[:, :cols]
        self.fresh = self.flat[shift:]
        if data is not None:
            self.view.copy_(data)

    def data_ptr(self):
        return self.fresh.data_ptr()

    def unmarked(self):
        """Whether anything beside the rows' values was written."""
        bytes_ = self.bytes.clone()
        dtype = self.flat.dtype
        rest = bytes_.view(dtype)
        size = rest.element_size()
        rest[self.shift:self.shift + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = (
            torch.full((size,), MARK, dtype=torch.uint8, device="cuda").view(dtype)[0])
        return bool((bytes_ != MARK).any())


def marked(dtype):
    """The value that a matrix holds before it is written."""
    size = torch.empty(0, dtype=dtype).element_size()
    return torch.full((size,), MARK, dtype=torch.uint8, device="cuda").view(dtype)[0]


def generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen
