"""Bounds for every single output of a matrix product (test infrastructure: plain torch only; tests/matmul_ref.py has the number formats).

The product of e4m3 operands on the matrix pipe, for 16-bit outputs: 8 products p of consecutive k are cut towards zero below 2^(E - 13), 2^E at most
the largest of them.  Two bounds on what that costs an output, both of which hold:
  at worst     a cut loses less than 2^-13 of the largest product of its 8, so a group loses less than 2^-10 of it.  The sum of the groups'
               largest products is at most  max|x| . max|w|  over the groups, and at most  |x| . |w|.
  in the mean  a cut is 0 .. 2^-13 of the largest product, half of that on average, towards zero.  Where all products have one sign, a group's eight
               such halves stand beside a sum of at least its largest product: 2^-11 of the result.  With random signs the cuts add up in squares: K of
               at most 2^-13 * P, P^2 <= the group's sum of squares, so sqrt(8) * 2^-13 * sqrt(sum p^2) = 2^-11.5 * sqrt(sum p^2) if every cut were the
               whole step; a uniform one spreads by 0.29 of it, so 2^-9.5, four times as much, stands for 14 standard deviations.
Signs that are random are part of the second bound: inputs without are held to the first alone (worst=True).
"""
import torch


def product_bound(x, w, dtype, fp8, worst=False):
    """(x @ w.T in float64, what an output of `dtype` may be off by): x, w the operands' values in float64; fp8: products of the e4m3 pipe."""
    ref, size = x @ w.t(), x.abs() @ w.abs().t()
    k = x.shape[1]
    # 128 products (64 of 16 bits) summed inside the matrix pipe with at most 2^-23 each, two more roundings per block, the scales' product
    off = (2 * min(k, 128) + 3 * -(-k // 64) + 8) * 2.0 ** -24 * size
    if fp8:
        xg, wg = (torch.nn.functional.pad(t, (0, -k % 8)).view(t.shape[0], -1, 8).abs().amax(2) for t in (x, w))
        cut = 2.0 ** -10 * torch.minimum(xg @ wg.t(), size)
        if not worst:
            cut = torch.minimum(cut, 2.0 ** -11 * ref.abs() + 2.0 ** -9.5 * ((x * x) @ (w * w).t()).sqrt())
        off = off + cut
    tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0
    return ref, torch.finfo(dtype).eps / 2 * (ref.abs() + off) + off + tiny


def check_every(got, x, w, fp8=False, worst=False, what=""):
    """got = x @ w.T rounded once to its type, at every output."""
    if 0 in got.shape:
        return
    ref, bound = product_bound(x, w, got.dtype, fp8, worst)
    assert got.shape == ref.shape and torch.isfinite(got).all(), what
    off = (got.double() - ref).abs()
    assert (off <= bound).all(), (what, (off / bound.clamp_min(1e-300)).max(), (off > bound).nonzero()[:4])
