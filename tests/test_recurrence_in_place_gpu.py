"""States updated in place where a cut between two streams goes through a chunk.

That chunk's map is worked out twice, by the stream that ends with it and by the
one that begins behind it, and both publish it in the same word of the
workspace.  The sequence that goes on behind the chunk may be finished, and its
state overwritten, before the second of them has run, so neither may read that
state from where it is updated: a word must hold the map of the state that the
call was given, whichever tile wrote it last.

The test reads the words back after the call and compares them with the states
of a call that is not in place.  The second part runs the same on the debug
build, which holds the map-only tiles back until the others have finished."""
import importlib
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent
ROWS, GROUP, STREAMS = 64, 8, 32

LENGTHS = [
    [90, 700, 333, 256, 111, 65, 1000, 64, 40, 450],
    [100] * 40,
    [37, 5, 300] * 12,
    [64 * 3 + 1, 130] * 10,
]


def cut_chunks(cu, chunks):
    """The chunks that a cut goes through: where the next sequence behind an even
    share of the chunks starts inside a chunk."""
    cut = set()
    prev = 0
    for i in range(1, STREAMS):
        share = chunks * i // STREAMS * ROWS
        row = next((int(s) for s in cu[:-1] if s >= share), chunks * ROWS)
        first = -(-row // ROWS)
        if prev < first < chunks:
            prev = first
            if row % ROWS and first * ROWS not in cu[:-1].tolist():
                cut.add(first - 1)
    return cut


def published(ws, chunks, D, chunk):
    """(A, H) of the map that a chunk of one tile of 64 channels published."""
    width = -(-D // 128) * 128
    start = 2048 + (8 + 4 * STREAMS) * width + (4 * (chunks + 1) + 15) // 16 * 16 + -ws.data_ptr() % 1024
    words = ws[start + 8 * chunk * 64:start + 8 * (chunk + 1) * 64].cpu().clone().view(torch.float32).view(64, 2)
    return words[:, 0], words[:, 1]


def check(gdn, lens, pool):
    D = 64
    cu = torch.tensor([0, *lens], dtype=torch.int64).cumsum(0)
    T, N = int(cu[-1]), len(lens)
    chunks = -(-T // ROWS)
    g = torch.Generator().manual_seed(T)
    x, a, b = (torch.randn(T, D, generator=g).cuda() for _ in range(3))
    A_log, dt_bias = (torch.rand(D, generator=g) * 3 - 5).cuda(), (torch.randn(D, generator=g) * 0.1).cuda()
    state = torch.randn(N, D, generator=g).cuda()
    want, want_final = gdn.recurrence.run(x, state, A_log, a, dt_bias, b, cu.cuda())
    out = torch.empty_like(x)
    ws = gdn.recurrence.alloc_workspace(T, D, "cuda")
    if pool:
        slots = torch.randperm(N + 2, generator=g)[:N].to(torch.int32).cuda()
        states = torch.zeros(N + 2, D, device="cuda")
        states[slots.long()] = state
        gdn.recurrence.run_pool_into(x, states, slots, A_log, a, dt_bias, b, cu.cuda(), out, ws)
        final = states[slots.long()]
    else:
        final = state.clone()
        gdn.recurrence.run_into(x, final, A_log, a, dt_bias, b, cu.cuda(), out, final, ws)
    assert torch.equal(out, want) and torch.equal(final, want_final)
    # a cut chunk is one map (not the last of a group of 8) that restarts, so its
    # constant is the state behind its last row: fp32, and so that row of `out`
    looked = 0
    for chunk in cut_chunks(cu, chunks):
        if chunk % GROUP == GROUP - 1:
            continue
        A, H = published(ws, chunks, D, chunk)
        assert bool((A < 0).all()), chunk
        assert torch.equal(H, want[chunk * ROWS + ROWS - 1].cpu()), chunk
        looked += 1
    assert looked >= 2
    assert gdn._native.read_device_status() == 0


@pytest.mark.parametrize("lens", LENGTHS, ids=lambda v: f"n{len(v)}")
@pytest.mark.parametrize("pool", [False, True])
def test_words_of_cut_chunks(gdn, lens, pool):
    gdn._native.read_device_status()
    for _ in range(3):
        check(gdn, lens, pool)


def test_words_of_cut_chunks_where_map_only_tiles_come_last():
    sys.path.insert(0, str(ROOT / "track-c-gdn_b200"))
    try:
        import build as native_build
    finally:
        sys.path.pop(0)
    lib = native_build.build(debug=True)
    res = subprocess.run([sys.executable, __file__], cwd=ROOT, env=dict(os.environ, GDN_B200_LIBRARY=str(lib)),
                         capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stdout[-3000:] + res.stderr[-3000:]
    assert "in place ok" in res.stdout, res.stdout[-2000:]


if __name__ == "__main__":
    sys.path.insert(0, str(ROOT))
    package = importlib.import_module("track-c-gdn_b200")
    assert package._native.LIB_PATH.name == "libgdn_b200_debug.so", package._native.LIB_PATH
    for lengths in LENGTHS:
        for in_pool in (False, True):
            check(package, lengths, in_pool)
    print("in place ok")
