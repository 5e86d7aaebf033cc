"""Serving operators called from several host threads at once, each on a stream
of its own, from their first launches in a process on: the C++ binding, the
calls' tags and the per-device settings are shared by all of them."""

import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]

_SCRIPT = textwrap.dedent(
    """
    import threading, torch
    from ninetoothed_b200 import programs
    from ninetoothed_b200.runtime import device_status

    gen = torch.Generator("cuda").manual_seed(5)
    def randn(*s):
        return torch.randn(s, generator=gen, device="cuda").half()
    def index(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    lens = [900, 3, 260]
    qkv = randn(sum(lens), 12, 128)
    q, k, v = qkv.split((8, 2, 2), 1)
    offsets, past, lengths = index([0, 900, 903, 1163]), index([0, 0, 0]), index(lens)
    table = index([[57 * s + c for c in range(57)] for s in range(3)])
    cos, sin = programs.rotary_tables(1024, 128, device="cuda")
    positions = torch.arange(sum(lens), dtype=torch.int32, device="cuda") % 1024
    drafts = randn(3, 4, 8, 128)

    def work():
        caches = [torch.zeros(171, 2, 16, 128, dtype=torch.int8, device="cuda") for _ in range(2)]
        scales = [torch.zeros(171, 2, device="cuda") for _ in range(2)]
        query, key = programs.paged_append(k, v, offsets, past, table, *caches, *scales, query=q, cos=cos, sin=sin,
                                           return_key=True)
        return [
            query, key, *caches, *scales,
            programs.rotary(q, cos, sin, positions, adjoint=True),
            *programs.prompt_attention(query, key, v, offsets, return_lse=True),
            *programs.paged_attention(drafts, *caches, *scales, table, lengths, return_lse=True),
        ]

    threads, results, errors = 4, {}, []
    start = threading.Barrier(threads)
    torch.cuda.synchronize()

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                start.wait()  # every thread's first launches race
                outs = [work() for _ in range(10)]
            stream.synchronize()
            results[i] = outs
        except Exception as exc:  # reported below
            errors.append(repr(exc))

    pool = [threading.Thread(target=run, args=(i,)) for i in range(threads)]
    for t in pool:
        t.start()
    for t in pool:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    expected = work()
    torch.cuda.synchronize()
    for i in range(threads):
        for outs in results[i]:
            for got, ref in zip(outs, expected):
                assert torch.equal(got, ref)
    assert device_status() == 0
    print("threads ok")
    """
)


def test_serving_calls_from_host_threads():
    proc = subprocess.run(
        [sys.executable, "-c", _SCRIPT], cwd=ROOT, capture_output=True, text=True, timeout=300
    )
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-4000:]
    assert "threads ok" in proc.stdout
