"""The 4-bit quantizer under torch's default types that loaders of 16-bit models set: the weight is the same, in every bit."""

import pytest
import torch


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("symmetric", [False, True])
def test_the_default_type_means_nothing(default, dtype, symmetric):
    from decik_amd.int4 import dequantize_int4, quantize_int4
    from decik_amd.rope import scaled_frequencies

    w = (torch.randn((9, 300), generator=torch.Generator().manual_seed(1)) * 0.02).to(dtype)
    scaling = dict(rope_type="longrope", short_factor=[1.1] * 32, original_max_position_embeddings=4096, factor=4.0)

    def made():
        q = quantize_int4(w, 64, symmetric)
        return q.packed, q.meta, dequantize_int4(q), scaled_frequencies(64, 1e6, scaling)[0]

    want = made()
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = made()
    finally:
        torch.set_default_dtype(before)
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(got, want))
