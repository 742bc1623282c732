"""CPU: sizes at which the operators' own arithmetic would wrap, refused before a device is touched."""

def quantise(features, sums=4096):
    import ltq
    return ltq.lib().ltq_quantize_tokens_u8(4096, 2, 1, features, features, 4096, 4096, sums, 0, None)

def test_code_sums_that_would_not_fit():
    """255 * 8421504 is the last multiple below 2^31."""
    import torch
    import ltq
    assert quantise(8421505) == -6 and "sum" in ltq.last_error()
    assert quantise((1 << 31) - 1) == -6
    if not torch.cuda.is_available():   # accepted: the next thing missing is the device
        assert quantise(8421504) == -3
        assert quantise((1 << 31) - 1, None) == -3
