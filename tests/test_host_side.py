"""The host side of the paged entries without a GPU: what they allocate, free,
order and launch, read from the log of a HIP runtime that does nothing else
(fake_hip.cpp). Each test runs in a process of its own that loads that runtime
ahead of the backend and never imports torch."""
import os
import subprocess
import sys
import textwrap

import pytest

import aigpu

HERE = os.path.dirname(os.path.abspath(__file__))
PACKAGE = os.path.dirname(os.path.dirname(os.path.abspath(aigpu.__file__)))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

PRELUDE = """
import ctypes as C, sys, threading
sys.modules["torch"] = None
fake = C.CDLL({fake!r}, mode=C.RTLD_GLOBAL)
fake.fake_log.restype = C.c_char_p
sys.path.insert(0, {package!r})
import aigpu
assert aigpu.available(), aigpu.last_error()
PTR, PER_THREAD = 1 << 20, 2

def log():
    return fake.fake_log().decode().splitlines()

def names(lines):
    return [line.split()[0] for line in lines]

def decode(batch=1, heads=16, kv=8, dim=128, length=4096, stream=0, gate=0, ok=1):
    cache = aigpu.AiGpuPagedCache(keys=PTR, values=PTR, table=PTR, lengths=PTR, batch=batch, pages=1 << 20, pageSize=16,
                                  kvHeads=kv, dim=dim, tableWidth=1 << 16)
    args = aigpu.AiGpuPagedDecode(cache=cache, q=PTR, out=1 << 28, maxLength=length, heads=heads, outputGate=gate,
                                  stream=stream)
    got = aigpu.lib().aigpu_paged_decode(C.byref(args))
    assert got == ok, aigpu.last_error()

log()
"""


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("fake") / "libfake_hip.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__",
                    f"-I{ROCM}/include", os.path.join(HERE, "fake_hip.cpp"), "-o", path], check=True)
    return path


def _run(fake, body):
    code = PRELUDE.format(fake=fake, package=PACKAGE) + textwrap.dedent(body)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


def test_one_launch_one_scratch_a_stream(fake):
    """the log itself: a stream's first call allocates and clears, the next one only launches"""
    _run(fake, """
        decode(stream=64)
        first = log()
        assert names(first) == ["hipMalloc", "hipMemset", "hipDeviceSynchronize", "launch"], first
        assert "paged_attention_kernel" in first[-1] and first[-1].split()[1] == "64"
        decode(stream=64)
        assert names(log()) == ["launch"]
    """)


def test_calls_on_the_per_thread_stream_are_ordered(fake):
    """its handle names another stream in every thread, and the stream goes with its thread: a call waits for the one
    before it, and for its own work, on the host, so that none of it is left when the next one takes the scratch"""
    _run(fake, """
        for _ in range(3):
            t = threading.Thread(target=lambda: decode(stream=PER_THREAD))
            t.start()
            t.join()
        calls = [n for n in log() if n.split()[0] in ("wait", "launch", "record", "finish")]
        assert names(calls) == ["launch", "finish"] * 3 and calls[1::2] == [f"finish {PER_THREAD}"] * 3, calls
        # behind a call of another stream, and one of another stream behind it
        for s in range(128, 137):
            decode(stream=s)
        log()
        decode(stream=PER_THREAD)
        decode(stream=136)
        calls = [" ".join(n.split()[:2]) for n in log()]
        assert calls == ["finish", "launch 2", "finish 2", "launch 136", "record 136"], calls
        # where its wait is refused the event is left, for whichever call comes next
        fake.fake_fail(b"finish", 2)
        decode(stream=PER_THREAD)
        log()
        decode(stream=PER_THREAD)
        decode(stream=136)
        calls = [" ".join(n.split()[:2]) for n in log()]
        assert calls == ["finish", "launch 2", "finish 2", "launch 136", "record 136"], calls
        # streams of one meaning wait where the handle changes only
        decode(stream=136)
        assert names(log()) == ["launch", "record"]
        # where the wait for the call before is refused, that call is still to be waited for
        fake.fake_fail(b"finish", 1)
        decode(stream=PER_THREAD)
        log()
        decode(stream=137)
        assert [" ".join(n.split()[:2]) for n in log()] == ["wait 137", "launch 137", "record 137"]
    """)


def test_scratch_in_use_is_kept_when_the_wait_for_it_is_refused(fake):
    """a scratch too small for a call is freed only after the work that may use it has been waited for: where that
    is refused (another thread captures), the call fails, the scratch stays, and a later call grows it"""
    _run(fake, """
        for own in (True, False):       # a stream's own scratch, and the one that later streams share
            stream = 64 if own else 99
            if not own:
                for s in range(65, 74):
                    decode(stream=s)
            decode(stream=stream)
            log()
            fake.fake_fail(b"hipDeviceSynchronize", 1)
            decode(stream=stream, kv=1, dim=256, ok=0)
            assert "scratch" in aigpu.last_error(), aigpu.last_error()
            lines = log()
            assert "hipFree" not in names(lines) and "launch" not in names(lines), lines
            decode(stream=stream)       # with what it has
            assert "hipMalloc" not in names(log())
            decode(stream=stream, kv=1, dim=256)
            lines = names(log())
            assert lines.index("hipDeviceSynchronize") < lines.index("hipFree") < lines.index("launch"), lines
    """)


@pytest.mark.parametrize("heads,kv,dim,batch", [(16, 8, 128, 1), (32, 4, 128, 1), (16, 1, 256, 3), (12, 12, 64, 2)])
def test_a_growing_conversation_allocates_once(fake, heads, kv, dim, batch):
    """max_length follows the longest sequence, step by step: only the first call allocates or waits for the device,
    on a stream with a scratch of its own and on those that share one"""
    _run(fake, f"""
        def steps(stream):
            first = log()
            for length in range(1, 20000, 7):
                decode(heads={heads}, kv={kv}, dim={dim}, batch={batch}, length=length, stream=stream)
                if length == 1:
                    first = names(log())
            assert first.count("hipMalloc") == 1, first
            rest = set(names(log()))
            assert rest <= {{"launch", "record"}}, rest

        steps(64)
        for s in range(65, 72):
            decode(heads={heads}, kv={kv}, dim={dim}, stream=s)
        log()
        steps(99)
    """)


def test_one_scratch_serves_every_batch_of_a_model(fake):
    """other batches, lengths and windows of the same heads and dim fit the first call's scratch"""
    _run(fake, """
        decode(batch=1, length=1)
        log()
        for batch in (1, 2, 7, 31, 200, 1000):
            for length in (1, 31, 33, 700, 9000, 131072):
                decode(batch=batch, length=length)
        assert set(names(log())) == {"launch"}
    """)
