"""GPU: one layer used by several host threads at once, each with batch sizes of its own, on a stream of its own.  The layer keeps
tensor maps for the boxes of the batch sizes that it has met; a launch must not go out with another one's."""
import threading

import pytest

pytestmark = pytest.mark.gpu


def test_one_layer_in_several_threads(cuda):
    import ltq
    torch = cuda
    K, N = 1024, 1536
    g = torch.Generator().manual_seed(0)
    layer = ltq.FullyConnected_t.from_float((0.05 * torch.randn(N, K, generator=g)).cuda(), torch.randn(N, generator=g).cuda())
    # streaming (up to 16 rows), few tiles of many widths, pairs
    sizes = [[1, 24, 100, 700], [16, 40, 130, 2000], [9, 17, 64, 150], [33, 90, 77, 300]]
    xs = {m: torch.randn(m, K, generator=g).half().cuda() for batch in sizes for m in batch}
    want = {m: layer.forward(x).clone() for m, x in xs.items()}
    torch.cuda.synchronize()
    errors, start = [], threading.Barrier(len(sizes))

    def work(batch):
        try:
            torch.cuda.set_device(0)
            stream = torch.cuda.Stream()
            start.wait()
            with torch.cuda.stream(stream):
                for _ in range(60):
                    for m in batch:
                        got = layer.forward(xs[m])
                        stream.synchronize()
                        if not torch.equal(got, want[m]):
                            errors.append(m)
                            return
        except Exception as e:   # noqa: BLE001 (shown by the assertion below)
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=(batch,)) for batch in sizes]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    layer._handle.check()


def test_batch_sizes_in_turn_keep_their_maps(cuda):
    """More widths than there are slots, in turn: every call as the first of its size."""
    import ltq
    torch = cuda
    layer = ltq.FullyConnected_t.from_float((0.05 * torch.randn(2048, 2048)).cuda())
    xs = {m: torch.randn(m, 2048).bfloat16().cuda() for m in range(17, 160, 7)}
    want = {m: ltq.FullyConnected_t(layer.weight_ptr_, layer.weight_qparams_).forward(x) for m, x in xs.items()}
    for _ in range(3):
        for m, x in xs.items():
            assert torch.equal(layer.forward(x), want[m])
    layer._handle.check()
