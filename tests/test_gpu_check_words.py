"""GPU: an expired wait and a refused argument of a cache call are both reported, whichever came first."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wait_first", [True, False])
def test_neither_hides_the_other(cuda, wait_first):
    import ltq
    torch, L = cuda, ltq.lib()
    cache = ltq.KVCache.empty(2, 1, 16, 32)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    k = torch.randn(1, 1, 32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    steps = [lambda: L.ltq_selftest_bounded_wait(0, 2000, stream), lambda: cache.append(k, k, ints([[7]]), ints([1]), ints([0, 1]), 1)]
    cache.check()
    for step in steps if wait_first else steps[::-1]:
        step()
    assert L.ltq_device_check(0, stream) == -4 and "0x900" in ltq.last_error()
    assert L.ltq_device_check(0, stream) == -1 and "block id" in ltq.last_error()
    assert L.ltq_device_check(0, stream) == 0
