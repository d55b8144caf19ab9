"""Device arrays of any type, and bfloat16 on the host, for the tests of the
language-model operators."""
import ctypes

import numpy as np

from conftest import load_backend

tl = load_backend()
from tensor_lang_b200 import runtime as rt  # noqa: E402

BF16_STEP = 2.0 ** -8   # half a step of bf16, relative to the value
F32 = 1e-5              # the suite's tolerance for float32 norms, sums and softmax


def bf16_bits(a):
    """float array -> bf16 bit patterns, round to nearest even (NaN stays NaN)."""
    a = np.ascontiguousarray(a, dtype=np.float32)
    b = a.view(np.uint32)
    r = ((b + np.uint32(0x7FFF) + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def bf16_value(bits):
    return (np.asarray(bits, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32)


def rounded(a, dtype):
    """The values an array of this element type holds, in float64."""
    if a is None:
        return None
    a = np.asarray(a, dtype=np.float32)
    return (bf16_value(bf16_bits(a)) if dtype == "bf16" else a).astype(np.float64)


CODE = {"f32": rt.F32, "bf16": rt.BF16}


class Dev:
    """Device allocations of one test: ``put`` / ``new`` give pointers, ``get`` reads back."""

    def __init__(self):
        self.dev = rt.Device.get(0)
        self.stream = self.dev.stream
        self.held = {}

    def raw(self, nbytes):
        p = ctypes.c_void_p()
        rt.check(rt.lib().tl_malloc(ctypes.byref(p), max(int(nbytes), 16), self.stream))
        self.held[p.value] = int(nbytes)
        return p.value

    def bytes_to(self, ptr, a):
        a = np.ascontiguousarray(a)
        rt.check(rt.lib().tl_memcpy_h2d(ptr, a.ctypes.data, a.nbytes, self.stream))
        self.dev.sync()

    def put(self, a, dtype=None):
        """An array on the device; dtype "f32"/"bf16" for elements, None as it is."""
        if a is None:
            return None
        if dtype == "bf16":
            a = bf16_bits(a)
        elif dtype == "f32":
            a = np.ascontiguousarray(a, dtype=np.float32)
        p = self.raw(a.nbytes)
        if a.nbytes:
            self.bytes_to(p, a)
        return p

    def rows(self, a, dtype, ld=None, lead=0, fill=7.0):
        """A matrix with rows `ld` elements apart, `lead` elements into its
        allocation; the elements between hold `fill`.  (pointer, ld)"""
        r, c = a.shape
        ld = ld or c
        flat = np.full(lead + r * ld, fill, np.float32)
        flat[lead:].reshape(r, ld)[:, :c] = a
        return self.put(flat, dtype) + lead * (2 if dtype == "bf16" else 4), ld

    def new(self, n, dtype="f32", fill=np.nan):
        """An output of n elements that holds `fill` until it is written."""
        return self.put(np.full(int(n), fill, np.float32), dtype)

    def zeros(self, nbytes):
        return self.put(np.zeros(max(int(nbytes), 16), np.uint8))

    def get(self, ptr, shape, dtype="f32"):
        n = int(np.prod(shape))
        a = np.empty(n, np.uint16 if dtype == "bf16" else np.float32)
        rt.check(rt.lib().tl_memcpy_d2h(a.ctypes.data, ptr, a.nbytes, self.stream))
        self.dev.sync()
        return (bf16_value(a) if dtype == "bf16" else a).reshape(shape)

    def get_rows(self, ptr, r, c, ld, dtype, lead=0):
        """(the matrix, the elements between its rows)"""
        e = 2 if dtype == "bf16" else 4
        flat = self.get(ptr - lead * e, (lead + r * ld,), dtype)
        m = flat[lead:].reshape(r, ld)
        return m[:, :c], np.concatenate([flat[:lead], m[:, c:].ravel()])

    def free(self):
        for p in self.held:
            rt.lib().tl_free(p, self.stream)
        self.held = {}
        self.dev.sync()

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.free()


def close(got, ref, dtype, name, rel=F32, scale=None):
    """|got - ref| <= rounding of the type + rel * (|ref| + scale); scale is
    max|ref| unless given (an array for sums: the magnitudes summed)."""
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    if not ref.size:
        return
    fin = np.isfinite(ref)
    assert np.array_equal(np.isnan(ref), np.isnan(got)), f"{name}: NaN in other places"
    np.testing.assert_array_equal(got[~fin], ref[~fin], err_msg=name)
    if scale is None:
        scale = np.abs(ref[fin]).max() if fin.any() else 0.0
    tol = rel * (np.abs(ref) + scale)
    if dtype == "bf16":
        tol = tol + BF16_STEP * np.abs(ref) * (1 + rel) + BF16_STEP * tol
    bad = fin & ~(np.abs(got - ref) <= tol)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(got - ref) - tol, -1)), ref.shape)
        raise AssertionError(f"{name}: {int(bad.sum())} of {ref.size} off; worst at {i}: "
                             f"got {got[i]!r}, want {ref[i]!r}, allowed {np.broadcast_to(tol, ref.shape)[i]:.3g}")
