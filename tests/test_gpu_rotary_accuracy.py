"""GPU accuracy of the rotary angles' cosines and sines by themselves: a unit
vector's rotation is (cos, sin) with nothing added, in fp32."""
import numpy as np
import pytest

from gpu_util import dev_f32, dev_u32, host, say
from oracle import oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("high", [4096, 131072, 2 ** 24])
def test_small_cosines_and_sines_keep_their_bits(gpu, high, interleaved):
    """relative to the value, wherever the angle lies. Of the two functions of the first term of the reduced angle: two
    units in their last place (2 2^-23 of the value they have there, which is off the wanted one by the second term,
    at most pi 2^-25 < 2^-23), half a unit of the addition; of the angle: its product, the turns' product and constant,
    and the oracle's own product, half a step of 64 bits each, 4 2^-53 of it; of the second term's product and of what
    its first order leaves out: below 1e-13"""
    import torch
    dim, n = 128, 3001
    freqs = O.rotary_frequencies(dim, 1e6)
    positions = np.random.default_rng(high).integers(0, high, n).astype(np.uint32)
    x = np.zeros((n, 1, dim), np.float32)
    first = np.arange(0, dim, 2) if interleaved else np.arange(dim // 2)
    second = first + 1 if interleaved else first + dim // 2
    x[..., first] = 1.0
    out = torch.empty((n, 1, dim), device="cuda")
    say("rotary of unit vectors", high, interleaved)
    gpu.rotary(dev_f32(x), out, dev_f32(freqs), positions=dev_u32(positions), interleaved=interleaved)
    got = host(out).astype(np.float64)
    angle = positions[:, None].astype(np.float64) * freqs.astype(np.float64)
    for want, at in ((np.cos(angle), first), (np.sin(angle), second)):
        tol = (2 * 2.0 ** -23 + 2.0 ** -24) * (np.abs(want) + 2.0 ** -23) + 4 * 2.0 ** -53 * angle + 1e-13
        err = np.abs(got[:, 0, at] - want)
        assert (np.abs(want) < 1e-3).sum() > 20
        assert (err <= tol).all(), ((err / tol).max(), (err > tol).mean())
