"""qc_rope_init's YaRN frequencies on the CPU, every pair of them, against the formula
of include/qrope.h: pow, a logarithm and a few products in IEEE double, each off by a
few units in the last place, of which the ramp's division keeps the size."""
import math

import numpy as np
import pytest


def yarn(rot, base, f, ctx, fast=32.0, slow=1.0):
    def c(b):
        return rot * math.log(ctx / (2 * math.pi * b)) / (2 * math.log(base))

    low, high = max(math.floor(c(fast)), 0), min(math.ceil(c(slow)), rot - 1)
    out = []
    for i in range(rot // 2):
        w = math.pow(base, -2 * i / rot)
        g = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        out.append(w / f * g + w * (1 - g))
    return np.array(out), low, high


CASES = [(64, 1e7, 4.0, 131072, {}), (64, 1e4, 8.0, 8192, {}), (128, 5e5, 2.0, 8192, {}), (256, 1e7, 4.0, 32768, {}),
         (24, 1e4, 16.0, 4096, {}), (96, 1e6, 1.0, 32768, {}), (64, 1e4, 0.5, 8192, {}),
         (64, 1e4, 4.0, 8192, dict(beta_fast=16.0, beta_slow=2.0)), (128, 1e4, 4.0, 4096, dict(beta_fast=40.0, beta_slow=0.5)),
         (64, 1e4, 4.0, 8192, dict(beta_fast=8.0, beta_slow=8.0)),      # the ends meet but for the rounding
         (64, 1e4, 4.0, 8192, dict(beta_fast=1.0, beta_slow=32.0)),     # high below low
         (64, 1e4, 4.0, 50, {}),                                        # low clamped to 0
         (64, 1e4, 4.0, 3, {}),                                         # both ends below 0
         (16, 10.0, 4.0, 1 << 30, {}), (2, 1e4, 4.0, 8192, {})]         # high clamped to rot - 1


@pytest.mark.parametrize("rot,base,f,ctx,betas", CASES)
def test_every_yarn_frequency(qcache, rot, base, f, ctx, betas):
    r = qcache.Rope(rot, base=base, scaling=qcache.ROPE_YARN, factor=f, orig_ctx=ctx, **betas)
    want, low, high = yarn(rot, base, f, ctx, betas.get("beta_fast", 32.0), betas.get("beta_slow", 1.0))
    np.testing.assert_allclose(np.array(r.freq.inv_freq[: rot // 2]), want, rtol=1e-13, atol=0)
    assert r.freq.mscale == pytest.approx(0.1 * math.log(f) + 1 if f > 1 else 1.0, rel=1e-15)


def test_the_cases_reach_every_form_of_the_ramp():
    """Ramps with pairs inside them, meeting ends, reversed ends and both clamps."""
    ends = [yarn(rot, base, f, ctx, b.get("beta_fast", 32.0), b.get("beta_slow", 1.0))[1:] for rot, base, f, ctx, b in CASES]
    assert any(high - low > 4 for low, high in ends) and any(high < low for low, high in ends)
    assert any(0 <= high - low <= 1 for low, high in ends) and any(low == 0 for low, _ in ends)
    assert any(high == rot - 1 for (_, high), (rot, *_) in zip(ends, CASES)) and any(high <= 0 for _, high in ends)
