"""Streams that fork, give tokens back and grow while earlier calls still wait on the caller's stream: each call sees
the page table and the pages as they were when it was enqueued."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_chunk import D, HQ, PT, QKV, Cache, attend_oracle, attend_tolerance, i32, visible  # noqa: E402

BACKLOG = 100_000_000   # SM clock cycles, some 50 ms: the calls of a test are enqueued well within it


class Queue:
    """Attention calls enqueued on a stream that is still busy, each checked against the tokens it had to see."""

    def __init__(self, cache, stream):
        self.c, self.st, self.calls = cache, stream, []
        self.gen = torch.Generator(device="cuda").manual_seed(17)

    def prepare(self, n):
        """Inputs of n calls, so that nothing is allocated or copied behind the backlog."""
        self.ready = []
        for _ in range(n):
            q = torch.randn((7, HQ * D), device="cuda", generator=self.gen).to(torch.bfloat16)
            self.ready.append((q, torch.full_like(q, -77.0)))
        self.lists = {}

    def lists_of(self, slot, length, m):
        return self.lists.setdefault((slot, length, m), [i32([slot]), i32([0, m]), i32([length])])

    def attend(self, slot, length, want_kv, m=5):
        q, out = self.ready[len(self.calls)]
        d = self.lists[(slot, length, m)]
        self.c.dec.chunk_attend(0, 1, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), m, None, q.data_ptr(),
                                out.data_ptr(), self.st.cuda_stream)
        self.calls.append((q, out, length, want_kv, m))

    def check(self):
        for j, (q, out, length, (k, v), m) in enumerate(self.calls):
            want, mag = attend_oracle(q[:m].double().view(m, HQ, D), k[:length], v[:length], visible(length - m, m))
            over = (out[:m].double().view(m, HQ, D) - want).abs() > attend_tolerance(want, mag)
            assert not over.any(), (j, length, int(over.sum()))
            assert (out[m:] == -77).all()


def busy(stream):
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(BACKLOG)


@pytest.fixture(scope="module", autouse=True)
def kernels_loaded(pkg):
    """Every kernel of these tests has run once: a kernel's first launch waits for the device."""
    for kv in ("bf16", "e4i8"):
        with Cache(pkg, kv, [40], max_streams=2) as c:
            c.fill()
            s = c.dec.fork(c.streams[0], 40)
            q = Queue(c, torch.cuda.current_stream())
            q.prepare(1)
            q.lists_of(s, 40, 5)
            q.attend(s, 40, c.values(0, c.streams[0], 40))
            c.dec.truncate(s, 39)
            qkv, out = torch.zeros((1, 2, QKV), device="cuda"), torch.zeros((1, 2, HQ * D), device="cuda")
            c.dec.truncate(c.streams[0], 32)
            c.dec.kv_step([c.streams[0], s], qkv.data_ptr(), out.data_ptr())
            c.dec.sync()


@pytest.mark.parametrize("kv", ["bf16", "e4i8"])
def test_fork_attend_truncate_extend_without_waiting(pkg, kv):
    with Cache(pkg, kv, [75], max_streams=3, spare=12, max_context=128) as c:
        c.fill()
        dec, a, st = c.dec, c.streams[0], torch.cuda.Stream()
        base = [t.clone() for t in c.values(0, a, 75)]
        q = Queue(c, st)
        q.prepare(3)
        fork = 1                               # the slot that the fork will have
        for n in (75, 40):
            q.lists_of(fork, n, 5)
        q.lists_of(a, 75, 5)
        busy(st)
        assert dec.fork(a, 75, st.cuda_stream) == fork
        q.attend(fork, 75, base)
        dec.truncate(fork, 40, st.cuda_stream)  # inside a shared page: the fork's own copy takes its place
        q.attend(fork, 40, base)
        dec.truncate(fork, 0, st.cuda_stream)
        assert not st.query()                  # nothing has run yet
        dec.extend(fork, 60)                   # new entries in the same places
        q.attend(a, 75, base)
        dec.sync()
        q.check()
        assert dec.length(fork) == 60 and dec.pool_stats()[0] == 17 - 5 - 4


def test_truncates_around_an_attention_without_waiting(pkg):
    """Each truncate replaces a shared last page by a copy; the attention between them reads the first copy."""
    with Cache(pkg, "bf16", [64], max_streams=4, spare=12, max_context=96) as c:
        c.fill()
        dec, a, st = c.dec, c.streams[0], torch.cuda.Stream()
        base = [t.clone() for t in c.values(0, a, 64)]
        q = Queue(c, st)
        q.prepare(4)
        b, d = dec.fork(a, 64), dec.fork(a, 64)
        for s, n in ((b, 56), (b, 40), (b, 23), (d, 64)):
            q.lists_of(s, n, 5)
        busy(st)
        for n in (56, 40, 23):
            dec.truncate(b, n, st.cuda_stream)
            q.attend(b, n, base)
        dec.truncate(b, 0, st.cuda_stream)
        q.attend(d, 64, base)
        assert not st.query()
        dec.sync()
        q.check()
        assert [int(x) for x in dec.pages(a)] == [int(x) for x in dec.pages(d)] and dec.pool_stats()[0] == 12


def test_step_that_grows_then_truncate_and_close_without_waiting(pkg):
    """A KV step that opens a page, then a truncate of the same stream, a close of it and a new stream in its slot."""
    with Cache(pkg, "bf16", [64, 32], max_streams=2, spare=8, max_context=96) as c:
        c.fill()
        dec, (a, b), st = c.dec, c.streams, torch.cuda.Stream()
        gen = torch.Generator(device="cuda").manual_seed(5)
        qkv = torch.randn((1, 2, QKV), device="cuda", generator=gen)
        kept = c.pool.clone()
        outs = []
        for wait in (True, False):
            c.pool.copy_(kept)
            out = torch.full((1, 2, HQ * D), -77.0, device="cuda")
            if wait:
                torch.cuda.synchronize()
            else:
                busy(st)
            dec.kv_step([a, b], qkv.data_ptr(), out.data_ptr(), st.cuda_stream)
            if wait:
                dec.sync()
            for s, n in ((a, 64), (b, 32)):
                dec.truncate(s, n, st.cuda_stream)
            if wait:
                dec.sync()
            else:
                assert not st.query()
            outs.append(out)
        dec.close_stream(a)                    # waits for the step and the truncate
        assert st.query()
        assert dec.open() == a
        dec.extend(a, 96)
        dec.sync()
        assert torch.equal(outs[0], outs[1]) and not (outs[1] == -77).all(-1).any()
        assert dec.length(a) == 96 and len(dec.pages(a)) == 96 // PT


@pytest.mark.parametrize("taker", ["fork", "step"])
def test_pages_given_back_on_one_stream_and_taken_on_another(pkg, taker):
    """The taker's stream is idle, and its copy or token goes into a page that a waiting attention has yet to read."""
    with Cache(pkg, "bf16", [64, 40], max_streams=3, spare=0, max_context=80) as c:
        c.fill()
        dec, (a, b), st, other = c.dec, c.streams, torch.cuda.Stream(), torch.cuda.Stream()
        base_a, base_b = [[t.clone() for t in c.values(0, s, n)] for s, n in ((a, 64), (b, 40))]
        qkv, out = torch.zeros((1, 1, QKV), device="cuda"), torch.zeros((1, 1, HQ * D), device="cuda")
        q = Queue(c, st)
        q.prepare(1)
        q.lists_of(b, 40, 5)
        was = set(int(x) for x in dec.pages(b))
        busy(st)
        q.attend(b, 40, base_b)
        dec.truncate(b, 0, st.cuda_stream)
        if taker == "fork":
            s = dec.fork(a, 20, other.cuda_stream)
        else:
            dec.kv_step([a], qkv.data_ptr(), out.data_ptr(), other.cuda_stream)
            s = a
        assert int(dec.pages(s)[-1]) in was and not st.query()
        dec.sync()
        q.check()
        n = 20 if taker == "fork" else 64
        assert all(torch.equal(x[:n], y[:n]) for x, y in zip(c.values(0, s, n), base_a))


def test_decode_after_extend_needs_ids(pkg, synth, tiny_files):
    """The greedy id from before a chunk does not follow it: not in the stream, and not in a fork of it."""
    _, files = tiny_files
    path = files[("bf16", "one_plus")]
    x, _ = synth.prompt_rows(synth.read_gguf(path)["text.token_embd.weight"], 20, np.random.default_rng(3), audio_rows=8,
                             audio_start=4)
    rt = pkg.runtime_config(device=0, weight_dtype=pkg.BF16, kv_dtype=pkg.BF16, max_streams=2, max_context=64)
    with pkg.Decoder.from_gguf(path, rt) as dec:
        a = dec.open()
        first = int(dec.prefill([a], [x])[0])
        dec.extend(a, 0)
        dec.decode_step([a])
        dec.extend(a, 3)
        dec.truncate(a, 24)                    # everything accepted
        b = dec.fork(a, 24)
        for s in (a, b):
            with pytest.raises(pkg.QkvError) as ei:
                dec.decode_step([s])
            assert ei.value.code == 1 and dec.length(s) == 24
        ids = dec.decode_step([a, b], in_ids=[first, first])
        assert ids[0] == ids[1] and dec.decode_step([a]) is not None
