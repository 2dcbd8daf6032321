"""What the shared attention's entries keep between calls (tensor maps by address and shape, which kernels have their shared memory): many caches, and calls of several host
threads at once."""
import threading

import pytest
import torch

from mini_inference_b200.ops import CudaOps
from tests.test_shared_attention import BF16, F32, check, problem

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from mini_inference_b200.ops import get_ops
    return get_ops("cuda:0")


@gpu
def test_more_caches_than_maps_are_kept_for(ops, monkeypatch):
    monkeypatch.setattr(CudaOps, "SHARED_BYTES", {BF16: 0, F32: 0})
    q, k, v, meta = problem([(32, [33, 40, 50])], 4, 1, 64, 16, BF16, seed=2)
    want = ops.shared_prefix_attention(q, k, v, meta, 4, 1, 64, 0.1)
    check(ops, q, k, v, meta, 4, 1, 64, scale=0.1, got=want)
    n, step = k.numel(), 8 * 16                                    # caches 256 bytes apart
    room = torch.zeros(2, n + 1300 * step, dtype=BF16, device=k.device)
    for i in [*range(1300), 0, 700]:
        at = [r[i * step:i * step + n].view(k.shape) for r in room]
        at[0].copy_(k)
        at[1].copy_(v)
        assert torch.equal(ops.shared_prefix_attention(q, *at, meta, 4, 1, 64, 0.1), want)
    ops.check_errors()


@gpu
@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, BF16), (64, F32), (128, F32)])
def test_calls_of_several_threads(ops, monkeypatch, D, dtype):
    """Each thread on its own stream, with its own inputs."""
    monkeypatch.setattr(CudaOps, "SHARED_BYTES", {BF16: 0, F32: 0})
    inputs = [problem([(160, [161, 200, 300]), (64, [65 + i, 90])], 8, 2, D, 16, dtype, seed=i) for i in range(4)]
    torch.cuda.synchronize()
    got, streams = [None] * 4, [torch.cuda.Stream() for _ in range(4)]
    begin = threading.Barrier(4)

    def calls(i):
        begin.wait(30)
        with torch.cuda.stream(streams[i]):
            for _ in range(20):
                got[i] = ops.shared_prefix_attention(*inputs[i], 8, 2, D, 0.1)
    threads = [threading.Thread(target=calls, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    ops.check_errors()
    for (q, k, v, meta), out in zip(inputs, got):
        check(ops, q, k, v, meta, 8, 2, D, scale=0.1, got=out)
