"""The head's formulas in 64 bits, with how far off a kernel may be that multiplies 16-bit operands exactly and adds in 32.

U is half a step of the 16-bit type relative to a value.  A sum of n products on the tensor cores takes n / 16 additions, each off by
at most 2^-22 of the sum of the products' sizes (additions need not round to nearest, and align their sixteen products first)."""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
STEP = 2.0 ** -22


def product_bound(a, b):
    """Of a @ b.T in 64 bits, from the sizes of its terms."""
    return (a.shape[1] / 16 + 2) * STEP * (a.abs() @ b.abs().T)


class Loss:
    """`loss`, `log_norms`, and `grads(...)` with their bounds, for hidden states and a weight as they are."""

    def __init__(self, hidden, weight, targets, softcap=0.0):
        self.dtype = weight.dtype
        self.on = (targets >= 0) & (targets < weight.shape[0])
        self.h, self.w = hidden.double()[self.on], weight.double()
        self.t = targets.long()[self.on]
        z = self.h @ self.w.T
        self.dz = product_bound(self.h, self.w)
        self.slope = torch.ones_like(z)
        if softcap:
            th = torch.tanh(z / softcap)
            z, self.slope = th * softcap, 1 - th * th
            self.dz = self.dz + softcap * 2.0 ** -21  # tanh, its argument's rounding and the product
        self.z, self.softcap = z, softcap
        n = torch.logsumexp(z, 1) if z.numel() else z.new_zeros(z.shape[0])
        # exponentials 2^-22 off, their arguments' roundings, sums of a tile in 32 bits: 1e-5 of the sum
        most = self.dz.amax(1) if z.numel() else n
        self.norm, self.d_norm = n, most + 1e-5 + n.abs() * 2.0 ** -23
        picked = z.gather(1, self.t[:, None])[:, 0]
        rows = targets.shape[0]
        f64 = dict(dtype=torch.float64, device=hidden.device)
        self.log_norms, self.loss, self.d_loss, self.d_norms = (torch.zeros(rows, **f64) for _ in range(4))
        self.log_norms[self.on], self.loss[self.on] = n, n - picked
        self.d_norms[self.on] = self.d_norm
        self.d_loss[self.on] = self.d_norm + most + (n - picked).abs() * 2.0 ** -23

    def grads(self, grad_loss, grad_norms=None):
        """(grad_hidden, its bound, grad_weight, its bound)."""
        u = U[self.dtype]
        b = grad_loss.double()[self.on]
        a = b + (0 if grad_norms is None else grad_norms.double()[self.on])
        p = torch.exp(self.z - self.norm[:, None])
        hot = torch.zeros_like(p)
        hot.scatter_(1, self.t[:, None], 1.0)
        g = (a[:, None] * p - b[:, None] * hot) * self.slope
        # the probability is as far off as its exponent, the gradient is rounded once (up to 64 rows keep the remainders, rounded in turn);
        # fp16 ends 2^-38 below the largest factor
        factor = torch.maximum(a.abs(), b.abs())
        most = factor.max() if factor.numel() else 0.0
        dp = self.dz + self.d_norm[:, None] + 2e-5
        dg = (a[:, None].abs() * p * dp + 2.0 ** -22 * (a.abs() + b.abs())[:, None] * (p + hot)) * self.slope.abs() + g.abs() * u + most * 2.0 ** -37
        if self.softcap:
            dg = dg + (a[:, None].abs() * p + b[:, None].abs() * hot) * (2.0 ** -20 + 2 * dp / self.softcap)
        return self._joined(g, dg, u)

    def _joined(self, g, dg, u):
        rows = self.on.shape[0]
        gh = torch.zeros((rows, self.w.shape[1]), dtype=torch.float64, device=self.w.device)
        dh = torch.zeros_like(gh)
        gh[self.on] = g @ self.w
        # sums over the vocabulary: in pieces, and pieces in 32 bits
        dh[self.on] = dg @ self.w.abs() + (self.w.shape[0] / 16 + 18) * STEP * (g.abs() @ self.w.abs())
        gw = g.T @ self.h
        dw = dg.T @ self.h.abs() + (rows / 16 + 18) * STEP * (g.abs().T @ self.h.abs())
        tiny = 2.0 ** -24 if self.dtype == torch.float16 else 2.0 ** -130
        return gh, dh + (gh.abs() + dh) * u + tiny, gw, dw + (gw.abs() + dw) * u + tiny


def unpack(codes, scales, zeros):
    """The weight of packed codes in 64 bits, and what its sums are off by per size of a hidden state: (weight, sizes)."""
    vocab, half = codes.shape
    q = torch.stack([codes & 15, codes >> 4], 2).reshape(vocab, 2 * half).double()
    group = 2 * half // scales.shape[1]
    s = scales.double().repeat_interleave(group, 1)
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 1)
    return (q - z) * s, ((q - 8).abs() + (0.0 if zeros is None else (z - 8).abs())) * s.abs()


def logits(hidden, codes, scales, zeros=None):
    """(logits in 64 bits, bound of a kernel that sums groups and joins them in 32 bits)."""
    w, size = unpack(codes, scales, zeros)
    h = hidden.double()
    z = h @ w.T
    per = h.abs() @ size.T
    # a group's sum, the sum of its hidden states, their product with the zero point, the scale, and the groups' sum
    groups = scales.shape[1]
    return z, (128 / 16 + 128 + 8 + groups) * 2.0 ** -23 * per
