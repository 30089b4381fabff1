"""Forward error analysis for the operator tests, in fp64 on the GPU: a value with a bound of its error, carried through matrix products
and roundings.  A test then holds a kernel's result to the bound of its own formula instead of to a number found by trying.

Rounding to a type is off by at most half a step: 2^-11 relative for fp16 (2^-25 absolute below its normal range), 2^-24 for fp32.  A
matrix product accumulates in fp32: every term may be added with an error of up to 2^-23 (the tensor core may cut where fp32 rounds)
of the partial sum, one addition for each group of 8 terms and up to 64 for the joining of groups and pieces.  fp32 operands enter as two
TF32 terms each, of which the product keeps all but 2^-20."""
import torch


class Bounded:
    """value (fp64) and a bound of its error, elementwise"""

    def __init__(self, value, error=None):
        self.value = value.double()
        self.error = torch.zeros_like(self.value) if error is None else error

    @property
    def T(self):
        return Bounded(self.value.T, self.error.T)

    def rounded(self, dtype):
        if dtype == torch.float16:
            return Bounded(self.value, self.error * (1 + 2.0 ** -11) + self.value.abs() * 2.0 ** -11 + 2.0 ** -25)
        return Bounded(self.value, self.error * (1 + 2.0 ** -24) + self.value.abs() * 2.0 ** -24)

    def slack(self, relative):
        return Bounded(self.value, self.error + self.value.abs() * relative)

    def __add__(self, other):
        return Bounded(self.value + other.value, self.error + other.error).slack(2.0 ** -23)

    def scaled(self, factor):
        factor = torch.as_tensor(factor, dtype=torch.float64, device=self.value.device)
        return Bounded(self.value * factor, self.error * factor.abs()).slack(2.0 ** -22)

    def holds(self, got, dtype=None):
        want = self if dtype is None else self.rounded(dtype)
        off = (got.double() - want.value).abs()
        bad = ~(off <= want.error)
        assert not bool(bad.any()), "off by up to %g of the bound, %d of %d values outside" % (float((off / want.error).max()), int(bad.sum()), bad.numel())


def product(a, b, dtype):
    """a b for Bounded a [m, k] and b [k, n]"""
    k = a.value.shape[1]
    aa, bb = a.value.abs(), b.value.abs()
    gamma = (k / 8 + 64) * 2.0 ** -23 + (2.0 ** -20 if dtype == torch.float32 else 0.0)
    return Bounded(a.value @ b.value, a.error @ (bb + b.error) + aa @ b.error + gamma * ((aa + a.error) @ (bb + b.error)) + 2.0 ** -60)
