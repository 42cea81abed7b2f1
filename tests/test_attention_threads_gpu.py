"""Two threads at once, each on a stream of its own: positions and attention over another sequence keep nothing between calls that they could share."""
import threading

import pytest
import torch

from flodl_b200 import ops
from test_cross_attention_gpu import C, case  # noqa: F401

pytestmark = pytest.mark.gpu


def work(data, mask, stream):
    with torch.cuda.stream(stream):
        q, k, v, do = data
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        f = ops.rotary_frequencies(q.shape[-1], device="cuda")
        out = []
        for m in (mask, None):
            turned = ops.qk_norm_rotary((leaves[0], leaves[1][:, :q.shape[1]]), None, None, f)
            o = ops.cross_attention(turned[0], ops.rotary(leaves[1], f), leaves[2], m)
            out += [o, *torch.autograd.grad((o, turned[1]), leaves, (do, turned[1]))]
        return out


def test_two_threads(C):
    shapes = [(2, 100, 1400, 16, 8, 64), (70, 17, 600, 8, 8, 64), (2, 1, 9000, 4, 2, 128), (24, 130, 300, 8, 8, 128)]
    jobs = []
    for i, shape in enumerate(shapes):
        g = torch.Generator(device="cuda").manual_seed(i)
        jobs.append((case(*shape, seed=i), torch.rand(shape[0], shape[2], generator=g, device="cuda") < 0.6))
    streams = [torch.cuda.Stream() for _ in shapes]
    want = [work(*job, torch.cuda.current_stream()) for job in jobs]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        try:
            for _ in range(5):
                got = work(*jobs[i], streams[i])
                streams[i].synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
        except Exception as e:  # noqa: BLE001  (a thread's error is the test's)
            wrong.append((i, repr(e)))
    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong and C.read_status(0) == 0
