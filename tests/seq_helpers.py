"""Shared by the tests of the operators along a sequence: element types, tolerances, calls through the C ABI."""
import ctypes as C
import math

import torch

import recpulse_b200 as rpb

TYPES = {"float32": torch.float32, "float64": torch.float64, "float16": torch.float16, "bfloat16": torch.bfloat16}
CODE = {"float32": rpb.F32, "float64": rpb.F64, "float16": rpb.F16, "bfloat16": rpb.BF16}


def acc_type(dtype):
    return torch.float64 if dtype == "float64" else torch.float32


def unit(dtype):
    """Half a step of the type the sums are held in."""
    return 2.0 ** -53 if dtype == "float64" else 2.0 ** -24


def ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def overflowed(slack, dtype, *values):
    """`slack`, infinite where one of `values` is beyond the range of the type that sums and states are held in: it is stored
    as an infinity there, and what is computed from it says nothing about the exact value."""
    most = torch.finfo(acc_type(dtype)).max
    for v in values:
        slack = torch.where(v.abs() < most, slack, float("inf"))
    return slack


def close(got, ref, slack, what, stored=None):
    """|got - ref| <= half a step of the stored type at the value + slack, elementwise; `ref` and `slack` float64.  Half a
    step is relative to the value as rounded, which may be `slack` larger; below the type's normal range a step is fixed."""
    stored = stored or got.dtype
    info = torch.finfo(stored)
    got, ref = got.detach().double().cpu(), ref.double().cpu()
    slack = slack.double().cpu() if torch.is_tensor(slack) else torch.tensor(float(slack), dtype=torch.float64)
    unknown = ~torch.isfinite(slack).expand_as(ref)        # behind an overflow of the arithmetic (see overflowed)
    got, ref, slack = got.masked_fill(unknown, 0), ref.masked_fill(unknown, 0), slack.expand_as(ref).masked_fill(unknown, 0)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    allowed = info.eps / 2 * (ref.abs() + slack) + slack + info.tiny * info.eps
    off = (got - ref).abs()
    bad = ~(off <= allowed)
    # to nearest, a value half a step or more beyond the largest one of the type is stored as the infinity of its sign
    beyond = info.max + info.eps / 2 * 2.0 ** (math.frexp(info.max)[1] - 1)
    bad &= ~(got.isinf() & (got.sign() == ref.sign()) & (ref.abs() + slack >= beyond))
    if bad.any():
        i = int(torch.where(bad, off / allowed, torch.zeros_like(off)).nan_to_num(float("inf"), float("inf")).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; worst: got {got.flatten()[i]!r}, "
                             f"want {ref.flatten()[i]!r}, allowed {allowed.expand_as(off).flatten()[i]!r}")
