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


def test_no_number_of_sms_is_written_into_the_code():
    """The plans ask the device for it (ten times and twenty times 148 included)."""
    import glob
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for path in glob.glob(os.path.join(root, "light-tensor_b200", "csrc", "ltq_*.cu*")):
        if os.path.basename(path).startswith(("ltq_cache", "ltq_tokens", "ltq_gemm_small")):
            code = re.sub(r"//[^\n]*", "", open(path).read())
            numbers = {int(n) for n in re.findall(r"(?<![\w.])(\d+)(?:u|ull)?\b", code)}
            assert not [n for n in numbers if n and n % 148 == 0], path
