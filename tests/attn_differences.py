"""Gradients against central differences of the fp64 forward (attn_oracle.py),
one (batch entry, head) at a time, along the gradient itself: there the
derivative is the block's gradient norm, far above what roundings allow, so
that a gradient that is missing, turned or scaled wrongly cannot pass."""
import math

import attn_oracle as A

STEP = 1e-4
# Every tolerance has to be this far below its derivative.
LEAST = 10.0


def blocks(q, k, v, do, out, lse, grads, options, fail):
    """Calls fail(name, b, h, off, tolerance, derivative) for every block of
    grads = {"dq", "dk", "dv"} that is off by more than its tolerance:

    * the elements' bounds for gradients from the given out and lse;
    * out and lse are rounded: how far the oracle's own gradients from them
      and from the exact ones differ along the direction;
    * the differences' third order: a step twice as long shows it, being off
      by four times as much;
    * fp64: sums of n terms of size f, 2^-50 f, over the step.

    Returns the smallest ratio of a derivative to its tolerance."""
    exact, exact_lse, _, _ = A.forward(q, k, v, **options)
    given = A.backward(do, q, k, v, out, lse, **options)
    there = A.backward(do, q, k, v, exact, exact_lse, **options)
    dd, x = do.double(), [t.double() for t in (q, k, v)]
    size = float((dd * exact).abs().sum())
    ratio = math.inf
    for i, n in enumerate(("dq", "dk", "dv")):
        B, H = x[i].shape[:2]
        for b in range(B):
            for h in range(H):
                g = there[n][0][b, h]
                d = g / g.norm()
                slopes = []
                for step in (STEP, 2 * STEP):
                    ends = []
                    for e in (step, -step):
                        y = list(x)
                        y[i] = x[i].clone()
                        y[i][b, h] += e * d
                        ends.append(float((A.forward(*y, **options)[0] * dd).sum()))
                    slopes.append((ends[0] - ends[1]) / (2 * step))
                tol = float((given[n][1][b, h] * d.abs()).sum()) + \
                    abs(float(((given[n][0] - there[n][0])[b, h] * d).sum())) + \
                    abs(slopes[1] - slopes[0]) + 2.0 ** -50 * size / STEP
                off = abs(slopes[0] - float((grads[n][b, h].double() * d).sum()))
                ratio = min(ratio, abs(slopes[0]) / tol)
                if not off <= tol:
                    fail(n, b, h, off, tol, slopes[0])
    return ratio
