"""First calls from many threads at once, in a process of its own: each finds
the device, and the results are those of one call after the other."""
import importlib
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def test_first_calls_at_once():
    res = subprocess.run([sys.executable, __file__], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-3000:]
    assert "threads ok" in res.stdout


if __name__ == "__main__":
    import threading

    import torch

    sys.path.insert(0, str(ROOT))
    gdn = importlib.import_module("track-c-gdn_b200")
    T, D, N = 900, 64, 16
    x = torch.randn(T, D, device="cuda")
    p = torch.zeros(D, device="cuda")
    outs = [torch.empty_like(x) for _ in range(N)]
    finals = [torch.empty(1, D, device="cuda") for _ in range(N)]
    spaces = [gdn.recurrence.alloc_workspace(T, D, "cuda") for _ in range(N)]
    streams = [torch.cuda.Stream() for _ in range(N)]
    torch.cuda.synchronize()
    start, errors = threading.Barrier(N), []

    def call(i):
        try:
            start.wait()
            gdn.recurrence.run_into(x, None, p, x, p, x, None, outs[i], finals[i], spaces[i],
                                    stream=streams[i].cuda_stream)
        except Exception as e:      # noqa: BLE001  (reported below)
            errors.append(e)

    threads = [threading.Thread(target=call, args=(i,)) for i in range(N)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    want, want_final = gdn.recurrence.run(x, None, p, x, p, x)
    for out, final in zip(outs, finals):
        assert torch.equal(out, want) and torch.equal(final, want_final)
    assert gdn._native.read_device_status() == 0
    print("threads ok")
