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


def test_a_table_whose_positions_wrap():
    """width * block_tokens of 2^64 and a little more is not a short table."""
    from test_tokens_abi import append, attention
    import ltq
    L = ltq.lib()
    for width in (1 << 27, 1 << 31, 1 << 60, (1 << 60) + 1, (1 << 64) - 1):
        assert append(L, width=width) == attention(L, width=width) == -1, width


def test_a_softmax_scale_that_wraps_in_base_two():
    """The kernels work with scale * log2(e): it has to be finite too."""
    from test_tokens_abi import attention
    import ltq
    L = ltq.lib()
    for scale in (3e38, -3e38, float("inf"), float("nan")):
        assert attention(L, scale=scale) == -1 and "softmax scale" in ltq.last_error()
