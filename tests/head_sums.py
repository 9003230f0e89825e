"""What the sums of a block-scaled e4m3 product may be off by, for operands whose products have independent random signs.

With ``l2 = sqrt(sum of the products' squares)``, a sum over any subset of the products is within ``8 l2`` of zero, and a sum of
independent errors of mean zero and at most ``c_k`` each within ``8 sqrt(sum c_k^2)``, but for a chance of ``2 exp(-32) = 3e-14``
(Hoeffding's inequality).

- fp32 additions, each off by at most ``2 U`` (``U = 2^-24``; twice, should an instruction cut instead of round) of a partial sum.
  Across blocks: ``blocks + 32`` (waves or pieces), partial sums within ``8 l2``.  Inside a block at most 16 (its eights), partial
  sums within 8 of the block's own l2; over the blocks these add up to ``sqrt(blocks) l2`` (Cauchy and Schwarz).  A block's sum times its scales is
  another rounding of that size.
- narrow: the e4m3 instructions cut each product towards zero below ``2^-13`` of the largest of its eight, by the exponents (a
  subnormal counts as ``2^-6``): mean zero under random signs, ``sum c_k^2 <= 8 * 2^-26 * l2^2``.
- The bias adds one rounding, the result's type half a step.
"""

import torch

U = 2.0 ** -24


def dequantized(q, scales, block_rows, least=None):
    """The operand in 64 bits; with ``least`` its magnitudes, ``least`` at the least before scaling."""
    v = q.float().double()
    if least is not None:
        v = v.abs().clamp_min(least)
    return v * scales.float().double().repeat_interleave(block_rows, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]


def product(a, a_scales, b, b_scales, bias=None):
    """The product in 64 bits and its l2, on the operands' device."""
    y = dequantized(a, a_scales, 1) @ dequantized(b, b_scales, 128).t().contiguous()
    if bias is not None:
        y = y + bias.double()
    left, right = dequantized(a, a_scales, 1, 2.0 ** -6), dequantized(b, b_scales, 128, 2.0 ** -6)
    return y, ((left * left) @ (right * right).t().contiguous()).sqrt()


def tolerance(y, l2, inner, dtype, narrow):
    blocks = -(-inner // 128)
    off = U * (16 * (blocks + 32) + 264 * blocks ** 0.5) * l2 + 2 * U * y.abs()
    if narrow:
        off = off + 8 * 8 ** 0.5 * 2.0 ** -13 * l2
    half = torch.finfo(dtype).eps / 2
    return half * y.abs() + (1 + half) * off + (2.0 ** -25 if dtype == torch.float16 else 0)
