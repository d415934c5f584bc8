"""GPU: threads that call the library for one device, each on a stream of its own."""
import threading

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def in_thread(f):
    out = []

    def run():
        try:
            out.append(f())
        except Exception as e:  # noqa: BLE001 - raised below
            out.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if isinstance(out[0], Exception):
        raise out[0]
    return out[0]


def test_a_threads_stream_is_its_own(sdb):
    L = sdb.lib()
    mine, other = torch.cuda.Stream(), torch.cuda.Stream()
    try:
        assert L.sdb200_set_stream(mine.cuda_stream) == 0

        def elsewhere():
            before = L.sdb200_get_stream()  # no choice of its own yet: the last one of any thread
            assert L.sdb200_set_stream(other.cuda_stream) == 0
            return before, L.sdb200_get_stream()

        before, after = in_thread(elsewhere)
        assert before == mine.cuda_stream and after == other.cuda_stream
        assert L.sdb200_get_stream() == mine.cuda_stream
        assert in_thread(L.sdb200_get_stream) == other.cuda_stream
    finally:
        sdb.backend.bind_stream()


def test_older_calls_beside_the_calls_for_several_requests(sdb):
    """One thread runs norms, another projections with adapters and attention, on streams of their own."""
    be = sdb.backend
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    randn = lambda *s, t=BF16: torch.randn(s, generator=g, device="cuda").to(t)  # noqa: E731
    x, W, A, B = randn(700, 512), randn(640, 512), randn(3, 16, 512), randn(3, 640, 16)
    rows = torch.arange(700, device="cuda", dtype=torch.int32) % 4 - 1
    h, gamma = randn(4096, 1024, t=torch.float32), randn(1024, t=torch.float32)
    n = torch.tensor([700], device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()

    def several():
        y = be.linear_lora(x, W, A, B, rows, out_dtype=BF16).view(700, 10, 64)
        return be.attention_ragged(y[:, :8], y[:, 8:9], y[:, 9:], n * 0, n, n * 0, n, 700, 700, causal=True)

    def older():
        y = h
        for _ in range(3):
            y = be.rms_norm(y, gamma, 1e-6)
        return y

    jobs = (several, older)
    want = [f() for f in jobs]
    torch.cuda.synchronize()
    got, wrong = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()) as _:
                for _ in range(60):
                    got[i].append(jobs[i]())
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - shown below
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    be.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
