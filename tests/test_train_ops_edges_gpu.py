"""The training operators where calls come close to what they were not made for, through litnicelm_b200.training."""
import math
import threading

import pytest
import torch

from litnicelm_b200 import training

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def rand(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- two calls at once from two host threads --------------------------------------------------------------------------------------


def at_once(*calls):
    """Each call from its own thread and stream, all starting together; what they return."""
    gate, results = threading.Barrier(len(calls)), [None] * len(calls)

    def run(i):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.default_stream())
        try:
            with torch.cuda.stream(stream):
                gate.wait()
                results[i] = calls[i]()
        except Exception as e:  # for the assertion in the main thread
            results[i] = e
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return results


def test_small_matrices_of_two_sizes_from_two_threads():
    """Each size wants its own amount of shared memory of one kernel."""
    g = gen(1)
    sets = [rand(g, *shape) for shape in ((64, 64), (64, 4096), (20, 1000))]
    alone = [training.orthogonalise(x) for x in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        got = at_once(*(lambda x=x: [training.orthogonalise(x) for _ in range(400)] for x in sets))
        for a, results in zip(alone, got):
            assert not isinstance(results, Exception), results
            assert all(torch.equal(a, b) for b in results)
