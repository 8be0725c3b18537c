"""Shared helpers of the tests of the operators on sequences of tokens: matrices with padding and guard values on the
device, expectations in 64 bits, and what a rounding to each type may cost."""
import numpy as np
import torch

from daphne_b200 import lib as names

TYPES = {"f64": (torch.float64, names.F64), "f32": (torch.float32, names.F32), "f16": (torch.float16, names.F16),
         "bf16": (torch.bfloat16, names.BF16)}
ALL = list(TYPES)
GUARD = 77.0


def half_step(t: torch.dtype) -> float:
    """Largest relative error of one rounding to nearest."""
    return torch.finfo(t).eps / 2


def smallest(t: torch.dtype) -> float:
    """Half the distance of two subnormal values: what a rounding may cost below the smallest normal value."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def wide(t: torch.dtype) -> torch.dtype:
    return torch.float64 if t == torch.float64 else torch.float32


class Mat:
    """rows x cols of `values` inside a larger device buffer: `pad` columns behind every row, `shift` elements in front,
    guard values everywhere else."""

    def __init__(self, values, dtype, pad=0, shift=0):
        values = torch.as_tensor(np.asarray(values) if not isinstance(values, torch.Tensor) else values)
        self.rows, self.cols = values.shape
        self.ld = self.cols + pad
        self.shift = shift
        self.buf = torch.full((shift + max(self.rows, 1) * self.ld + 64,), GUARD, dtype=dtype, device="cuda")
        self.view = self.buf[shift:shift + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols]
        self.view.copy_(values.to(dtype))

    @staticmethod
    def empty(rows, cols, dtype, pad=0, shift=0):
        return Mat(torch.full((rows, cols), GUARD, dtype=torch.float64), dtype, pad, shift)

    @property
    def ptr(self):
        return self.buf.data_ptr() + self.shift * self.buf.element_size()

    @property
    def at(self):
        return self.ptr, self.ld

    def f64(self) -> np.ndarray:
        return self.view.double().cpu().numpy()

    def guards_intact(self) -> bool:
        mask = torch.ones_like(self.buf, dtype=torch.bool)
        mask[self.shift:self.shift + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = False
        return bool((self.buf[mask].double() == GUARD).all())


def stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def scratch(nbytes: int):
    return torch.full((max(int(nbytes), 16),), 0xFF, dtype=torch.uint8, device="cuda")


def assert_within(got: np.ndarray, exp: np.ndarray, bound: np.ndarray, what=""):
    """|got - exp| <= bound element by element; NaNs and infinities coincide."""
    assert got.shape == exp.shape, f"{what}: shape {got.shape} vs {exp.shape}"
    fin = np.isfinite(exp)
    assert np.array_equal(np.isnan(got), np.isnan(exp)), f"{what}: NaN pattern differs"
    assert np.array_equal(got[~fin & ~np.isnan(exp)], exp[~fin & ~np.isnan(exp)]), f"{what}: infinities differ"
    bound = np.broadcast_to(np.asarray(bound, dtype=np.float64), exp.shape)
    err = np.abs(got[fin] - exp[fin])
    bad = err > bound[fin]
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} outside, worst {np.max(err[bad] / np.maximum(bound[fin][bad], 1e-300)):.3g} "
                           f"times the bound, at {np.argwhere(fin)[np.argmax(bad)].tolist()}")
