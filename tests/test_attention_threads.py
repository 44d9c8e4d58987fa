"""One attention plan, several host threads."""
import os
import subprocess
import threading

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_what_a_forward_writes_is_atomic(tmp_path):
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    r = subprocess.run(["g++", "-std=c++17", "-fsyntax-only", f"-I{cuda}/include", os.path.join(ROOT, "tests", "plan_threads_check.cc")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.gpu
def test_calls_of_one_plan_from_two_threads():
    """Different kernels at once, each thread on a stream of its own; `kernel` names one of them all the while, and errors stay with their thread."""
    import torch

    import darknet_b200 as dn
    plan, done, wrong = dn.CrossAttentionPlan(8, 2, 64), threading.Event(), []
    D = lambda t: dn.as_tensor(t, dn.NHWC)  # noqa: E731

    def job(seed, dtype, lq, side):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                g = torch.Generator(device="cuda").manual_seed(seed)
                q = torch.randn((2, 1, lq, 512), generator=g, device="cuda").to(dtype)
                k, v = torch.randn((2, 2, side, side, 128), generator=g, device="cuda").to(dtype)
                y, first = torch.zeros_like(q), None
                for i in range(200):
                    if i % 50 == 7:
                        with pytest.raises(dn.DarknetB200Error, match=f"for queries of {seed}"):
                            plan.forward(D(q[:1].expand(seed, -1, -1, -1).contiguous()), D(k), D(v), D(torch.zeros((seed, 1, lq, 512), dtype=dtype, device="cuda")))
                    y.zero_()
                    plan.forward(D(q), D(k), D(v), D(y))
                    first = y.clone() if first is None else first
                    if not torch.equal(first, y):
                        wrong.append((seed, i))
            stream.synchronize()
        except BaseException as e:      # noqa: BLE001 -- the test's own thread reports it
            wrong.append(e)

    def look():
        while not done.is_set():
            if plan.kernel not in ("none", "rows_bf16", "tc_bf16", "rows_f32", "tc_f32"):
                wrong.append(plan.kernel)

    threads = [threading.Thread(target=job, args=a) for a in [(3, torch.bfloat16, 2, 19), (4, torch.bfloat16, 100, 19), (5, torch.float32, 70, 13)]]
    watcher = threading.Thread(target=look)
    watcher.start()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    done.set()
    watcher.join()
    torch.cuda.synchronize()
    plan.check_status()
    assert not wrong, wrong[:3]
