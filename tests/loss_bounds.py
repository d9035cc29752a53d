"""The definition of linear_cross_entropy's gradients in 64 bits, and how far results in bf16 may be from it.

A bf16 number has 8 bits, so rounding to it is off by 2^-8 of the value at most, and by 2^-8 / sqrt(3) = 2.3e-3 root mean square at
the worst mantissa.  Two such roundings: dz before the products (tokens of up to 64 in a call keep 16 bits instead: 2^-16), and the result.
The first counts relative to what is added up, not to the sum:

* an element is off by at most 2^-8 (sum |dz| |factor| + |sum|), and what the logits of the backward are off;
* the 2-norm of a block of many elements, errors of dz being independent, by 2.3e-3 (norm of sqrt(sum dz^2 factor^2) + norm of the block).

Logits of the backward: an accumulator loses up to 2^-23 of the sum of magnitudes S every 16 elements of the reduction; statistics a few
2^-22 in addition: a relative error of p of d = (H / 16 + 8) 2^-22 S + 2^-18.  The sums over V and T: (K / 16 + 8) 2^-23 of the magnitudes."""
import torch

U = 2.0 ** -8
RMS = U / 3 ** 0.5


class Gradients:
    """``dx``, ``dw`` exactly; ``*_abs``: sums of magnitudes; ``*_rss``: roots of sums of squares."""

    def __init__(self, x, w, y, scale, ignore=-100):
        T, H = x.shape
        V = w.shape[0]
        x, w = x.detach().double(), w.detach().double()
        live = y != ignore
        z = x @ w.t()
        p = (z - torch.logsumexp(z, 1, keepdim=True)).exp()
        dz = p.clone()
        dz[torch.arange(T, device=x.device), y.clamp(min=0)] -= 1.0
        c = (scale.double() * live).unsqueeze(1)
        dz, p = dz * c, p * c.abs()
        self.dx, self.dw = dz @ w, dz.t() @ x
        first = 2.0 ** -16 if T <= 64 else U
        d = (H / 16 + 8) * 2.0 ** -22 * float((x.abs() @ w.abs().t()).max()) + 2.0 ** -18
        err = (first + (max(T, V) / 16 + 8) * 2.0 ** -23) * dz.abs() + d * p
        self.dx_worst, self.dw_worst = err @ w.abs(), err.t() @ x.abs()
        self.dx_rss, self.dw_rss = ((dz.square() @ w.square()).sqrt(), (dz.square().t() @ x.square()).sqrt())
        self.first_rms, self.d = first / 3 ** 0.5, d

    def check(self, gx, gw):
        """Every element, and the norms of both."""
        for got, want, worst, rss in ((gx, self.dx, self.dx_worst, self.dx_rss), (gw, self.dw, self.dw_worst, self.dw_rss)):
            if got is not None:
                check_elements(got, want, worst)
                self.check_norm(got, want, rss, worst)

    def check_norm(self, got, want, rss, worst):
        """(``worst`` bounds blocks of so few elements that a mean square says nothing.)"""
        assert torch.isfinite(got).all()
        off = float((got.double() - want).norm())
        limit = RMS * float(want.norm()) + (self.first_rms + self.d) * float(rss.norm()) if want.numel() >= 1000 else float((worst + U * want.abs()).norm())
        assert off <= limit * 1.001 + 1e-30, (off, limit)


def check_elements(got, want, worst):
    off = (got.double() - want).abs() - (worst + U * (want.abs() + worst))
    assert float(off.max()) <= 1e-30, (float(off.max()), int(off.argmax()))
