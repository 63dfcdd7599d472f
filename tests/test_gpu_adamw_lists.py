"""Lists at the limits of a launch, tensors of 16 bits with memory of others between them, clipping with many partial sums."""

import math

import numpy as np
import pytest
import torch

import _adamw_oracle as O
from emerging_optimizers import hip_kernels as k
from test_gpu_adamw import BF16, F16, F32, HYPER, check_update, moments, np64, packed_like, snapshot, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [66, 67, 140])
@pytest.mark.parametrize("bits", [32, 8])
def test_as_many_tensors_with_copies_as_a_launch_takes_and_more(gpu, bits, count):
    gen = torch.Generator().manual_seed(71)
    sizes = [1 + 37 * i % 300 for i in range(count)]
    params, grads, model = values(gen, sizes, 0.02), values(gen, sizes, 1e-3, BF16, offset=1), values(gen, sizes, 1.0, BF16, offset=3)
    ms, vs = moments(gen, sizes)
    if bits == 8:
        ms, vs = packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")
    before = snapshot(params, ms, vs, bits)
    update = k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit
    update(params, grads, ms, vs, step=3, model_params=model, **HYPER)
    check_update(params, grads, ms, vs, before, method="decoupled", step=3, bits=bits, model=model)


class Spaced:
    """Tensors in one buffer, ``gap`` elements of nobody's before each and behind the last."""

    def __init__(self, gen, sizes, scale, dtype, gap, square=False):
        self.gap, self.sizes = gap, sizes
        self.flat = torch.full((sum(sizes) + gap * (len(sizes) + 1),), 5.0, dtype=dtype)
        self.at = np.cumsum([gap] + [n + gap for n in sizes])[:-1].tolist()
        for a, n in zip(self.at, sizes):
            x = torch.randn(n, generator=gen) * scale
            self.flat[a : a + n] = (x * x if square else x).to(dtype)
        self.flat = self.flat.to("cuda")
        self.tensors = [self.flat[a : a + n] for a, n in zip(self.at, sizes)]

    def untouched(self):
        owned = torch.zeros(self.flat.numel(), dtype=torch.bool)
        for a, n in zip(self.at, self.sizes):
            owned[a : a + n] = True
        return bool((self.flat.cpu()[~owned] == 5.0).all())


@pytest.mark.parametrize("types", [(BF16, BF16, None), (F16, F16, None), (BF16, F32, None), (F32, BF16, BF16), (F32, F16, F16), (F32, F32, BF16)], ids=str)
@pytest.mark.parametrize("bits, rounding", [(32, None), (8, "nearest"), (8, "dithered")])
def test_memory_between_tensors_of_16_bits_stays_as_it_was(gpu, bits, rounding, types):
    p_type, g_type, low = types
    gen = torch.Generator().manual_seed(72)
    sizes = [5, 64, 4099, 70, 1, 1023, 130]
    for gap in (1, 7, 8):
        params, grads = Spaced(gen, sizes, 0.02, p_type, gap), Spaced(gen, sizes, 1e-3 if g_type != F16 else 1.0, g_type, gap)
        m, v = Spaced(gen, sizes, 1e-3, F32, gap), Spaced(gen, sizes, 1e-3, F32, gap, square=True)
        copies = None if low is None else Spaced(gen, sizes, 1.0, low, gap)
        ms, vs = m.tensors, v.tensors
        if bits == 8:
            ms, vs = packed_like(ms, "exp_avg"), packed_like(vs, "exp_avg_sq")
        update = k.fused_adamw_update if bits == 32 else k.fused_adamw_update_8bit
        step = 3  # (dithered codes are to nearest until the fifth step)
        before = snapshot(params.tensors, ms, vs, bits)
        kept = grads.flat.clone()
        model = None if copies is None else copies.tensors
        update(params.tensors, grads.tensors, ms, vs, step=step, model_params=model, **({"rounding": rounding} if rounding else {}), **HYPER)
        check_update(params.tensors, grads.tensors, ms, vs, before, method="decoupled", step=step, bits=bits, model=model)
        assert torch.equal(grads.flat, kept)
        norm = k.clip_grads_by_global_norm(grads.tensors, max_norm=1e-4)
        assert float(norm) > 1e-4
        for which, packed in (("exp_avg", ms), ("exp_avg_sq", vs)) if bits == 8 else ():
            k.unpack_moments_8bit(packed, params.tensors, which=which)
        for part in (params, grads, m, v, copies):
            assert part is None or part.untouched()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_clipping_and_scaling_with_many_partial_sums_at_odd_places(gpu, dtype):
    """More partial sums than the scaling kernel adds up itself: the factor comes ready from a launch of its own."""
    gen = torch.Generator().manual_seed(73)
    sizes = [1 + 53 * i % 400 for i in range(700)] + [33333]
    for gap in (1, 3):
        grads = Spaced(gen, sizes, 0.5, dtype, gap)
        raw = [np64(g) for g in grads.tensors]
        exact = math.sqrt(sum(float((g**2).sum()) for g in raw))
        norm = k.clip_grads_by_global_norm(grads.tensors, max_norm=0.75)
        assert abs(float(norm) - exact) <= 1.01 * O.U * exact
        want = 0.75 / (exact + 1e-6)
        for g, b in zip(grads.tensors, raw):
            O.assert_within(np64(g), b * want, O.to_type(b * want, 8 * O.U * abs(b * want), dtype) + 1e-300, "clipped")
        assert grads.untouched()
        raw = [np64(g) for g in grads.tensors]
        k.scale_tensors(grads.tensors, torch.tensor(1.7, device=gpu))
        f = float(np.float32(1.7))
        for g, b in zip(grads.tensors, raw):
            O.assert_within(np64(g), b * f, O.to_type(b * f, O.U * abs(b * f), dtype) + 1e-300, "scaled")
        assert grads.untouched()
