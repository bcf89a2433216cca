"""Values at the edge of what the chunk operators take: vectors with scale zero, queries that are not finite, moves
between streams that share pages."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_chunk import (D, HKV, HQ, PT, QKV, Cache, append_oracle, attend_oracle,  # noqa: E402
                            attend_tolerance, check_attend, i32, raw, run_attend, run_move, visible)

# rows of one call: up to 16, up to 64 and up to 128 at a time take three paths through the kernel; the long contexts
# are cut between SMs, the short ones are not
CHUNKS = [(3, 9), (900, 14), (5, 40), (1300, 60), (10, 100), (700, 128)]


def layout(chunks):
    return [b + m for b, m in chunks], [sum(m for _, m in chunks[:j]) for j in range(len(chunks) + 1)]


def queries(rows, seed=2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (1.3 * torch.randn((rows, HQ * D), device="cuda", generator=gen)).to(torch.bfloat16)


@pytest.mark.parametrize("kv", ["fp8", "e4i8"])
@pytest.mark.parametrize("masked", [False, True])
def test_attend_vectors_with_scale_zero(pkg, kv, masked):
    """Keys and values of scale 0, visible and hidden, among them the first and the last token of each chunk."""
    chunks = [c for c in CHUNKS if c[1] <= 64] if masked else CHUNKS
    lens, starts = layout(chunks)
    masks = None
    if masked:
        masks = [(0x9249249249249249 << (j % 3)) & ((1 << 64) - 1) if j % 5 else 0 for m in (c[1] for c in chunks) for j in range(m)]
    with Cache(pkg, kv, lens) as c:
        c.fill()
        for s, (base, m) in zip(c.streams, chunks):
            pages = c.dec.pages(s)
            for t in {0, 1, base // 2, base, base + 1, base + m // 2, base + m - 1}:
                page, at = int(pages[t // PT]), t % PT
                c.scales[0, page, :, :, at] = 0.0
                c.pool[0, page, 0, :, at] = 0 if t % 2 else 0x38      # code 0, or a code that the scale makes 0
        c.poison_behind(lens)
        q = queries(starts[-1])
        out = run_attend(c, chunks, q, starts, masks)
        check_attend(c, chunks, q, starts, out, masks)


@pytest.mark.parametrize("kv", ["bf16", "fp8", "e4i8"])
@pytest.mark.parametrize("masked", [False, True])
def test_attend_queries_that_are_not_finite(pkg, kv, masked):
    """NaN and infinite queries give NaN in their own row and head, as the formula does, and nothing elsewhere."""
    chunks = [c for c in CHUNKS if c[1] <= 64] if masked else CHUNKS
    lens, starts = layout(chunks)
    masks = [(1 << (j + 1)) - 1 if j % 7 != 3 else 0 for _, m in chunks for j in range(m)] if masked else None
    with Cache(pkg, kv, lens) as c:
        c.fill()
        c.poison_behind(lens)
        clean = queries(starts[-1])
        q = clean.clone().view(-1, HQ, D)
        hit = torch.zeros((starts[-1], HQ), dtype=torch.bool, device="cuda")
        for j, (base, m) in enumerate(chunks):
            k, _ = c.values(0, c.streams[j], base + m)
            for r, head, value in ((0, 3, "nan"), (1, 0, "first"), (m // 2, 8, "nan"), (m // 2, 15, "first"), (m - 1, 14, "last")):
                # infinity with the sign of one visible token's key: that score is +infinity
                token = 0 if value == "first" else base - 1
                inf = float("inf") if k[token, head // 2, 77] >= 0 else -float("inf")
                q[starts[j] + r, head, 77] = float("nan") if value == "nan" else inf
                hit[starts[j] + r, head] = True
        q = q.view(-1, HQ * D)
        out = run_attend(c, chunks, q, starts, masks)
        for j, (base, m) in enumerate(chunks):
            rows = slice(starts[j], starts[j + 1])
            k, v = c.values(0, c.streams[j], base + m)
            seen = visible(base, m, masks[rows] if masks else None)
            want, mag = attend_oracle(clean[rows].double().view(m, HQ, D), k, v, seen)
            got, bad = out[rows].double().view(m, HQ, D), hit[rows]
            assert torch.isnan(got[bad]).all(), (j, base, m)
            assert not ((got - want).abs() > attend_tolerance(want, mag))[~bad].any() and torch.isfinite(got[~bad]).all(), (j, base, m)


@pytest.mark.parametrize("kv", ["f32", "bf16", "e4i8"])
def test_tokens_move_between_streams_that_share_pages(pkg, kv):
    """Down within shared pages: as within one stream.  Up into them: reported, nothing moves.  Past them: any way."""
    with Cache(pkg, kv, [90], layers=2, max_streams=2, spare=8, max_context=128) as c:
        c.fill()
        dec, a = c.dec, c.streams[0]
        b = dec.fork(a, 70)                    # four shared pages, the fifth of its own
        dec.sync()
        before, sc = c.pool.clone(), c.scales.clone() if c.scales is not None else None
        for g in ((a, 3, b, 10, list(range(0, 30))), (a, 0, b, 1, [0]), (b, 20, a, 60, list(range(0, 20)))):
            with pytest.raises(pkg.QkvError) as ei:
                run_move(c, [g])
            assert ei.value.code == 5
            assert torch.equal(raw(c.pool), raw(before)) and (sc is None or torch.equal(c.scales, sc)), g
        for src, from_base, dst, to_base, keep in ((a, 30, b, 10, list(range(0, 40, 2))), (b, 5, a, 0, list(range(0, 60))),
                                                   (a, 3, b, 64, [0, 2, 30, 61, 66])):
            want = [[t.clone() for t in c.values(1, s, 70)] for s in (a, b)]
            n, at = len(keep), [from_base + t for t in keep]
            for s, kv_of in ((a, want[0]), (b, want[1])):
                for x, y in zip(want[0 if src == a else 1], kv_of):
                    moved = x[at].clone() if s == dst else None
                    if s == dst:
                        y[to_base:to_base + n] = moved
            shared = 64                        # what one stream has there, the other has
            if to_base < shared:
                for x, y in zip(want[0 if dst == a else 1], want[1 if dst == a else 0]):
                    y[to_base:min(to_base + n, shared)] = x[to_base:min(to_base + n, shared)]
            run_move(c, [(src, from_base, dst, to_base, keep)])
            for s, kv_of in ((a, want[0]), (b, want[1])):
                for x, y in zip(c.values(1, s, 70), kv_of):
                    assert torch.equal(x, y), (src, dst, to_base)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_attend_one_chunk_of_many_rows(pkg, kv):
    """A whole prompt as one chunk, and a second one behind it: rows of every block against the oracle."""
    chunks = [(77, 9000), (0, 2500)]
    lens, starts = layout(chunks)
    with Cache(pkg, kv, lens) as c:
        c.fill()
        c.poison_behind(lens)
        q = queries(starts[-1])
        out = run_attend(c, chunks, q, starts)
        for j, (base, m) in enumerate(chunks):
            k, v = c.values(0, c.streams[j], base + m)
            rows = torch.arange(m % 61, m, 61, device="cuda")
            seen = torch.arange(base + m, device="cuda")[None] <= base + rows[:, None]
            want, mag = attend_oracle(q[starts[j] + rows].double().view(-1, HQ, D), k, v, seen)
            assert not ((out[starts[j] + rows].double().view(-1, HQ, D) - want).abs() > attend_tolerance(want, mag)).any(), j


@pytest.mark.parametrize("kv", ["fp8", "e4i8"])
@pytest.mark.parametrize("chunk", [True, False])
def test_append_of_vectors_near_the_end_of_the_range(pkg, kv, chunk):
    """8-bit caches: vectors of 1e-30 down to the smallest f32 and zeros among them; chunk_append and kv_append alike."""
    sizes = [1e-30, 1e-35, 1e-36, 1e-37, 1e-38, 1e-40, 1e-42, 1e-44, 0.0]
    n = len(sizes)
    with Cache(pkg, kv, [n]) as c:
        gen = torch.Generator(device="cuda").manual_seed(9)
        qkv = torch.randn((n, QKV), device="cuda", generator=gen)
        # k goes through the norm, which divides vectors this small by sqrt(eps): 1000 times as large
        qkv[:, HQ * D:] *= torch.tensor(sizes, device="cuda")[:, None]
        qkv[:, HQ * D::5] = 0.0
        slots, pos = i32([c.streams[0]] * n), i32(range(n))
        axes = torch.zeros((3, n), dtype=torch.int32, device="cuda")
        q = torch.empty((n, HQ * D), device="cuda")
        if chunk:
            c.dec.chunk_append(0, n, slots.data_ptr(), pos.data_ptr(), axes.data_ptr(), (64, 0, 0), False, qkv.data_ptr(),
                               q.data_ptr(), pkg.F32)
        else:
            axes = torch.stack([pos] * 3).contiguous()
            c.dec.kv_append(0, n, slots.data_ptr(), pos.data_ptr(), qkv.data_ptr(), q.data_ptr())
        c.dec.sync()
        want_k, mag = append_oracle(qkv[:, HQ * D:(HQ + HKV) * D].double().view(n, HKV, D),
                                    torch.tensor(c.kn[0], device="cuda").double(), axes, [0] * 64)
        want_v = qkv[:, (HQ + HKV) * D:].double().view(n, HKV, D)
        page = int(c.dec.pages(c.streams[0])[0])
        assert torch.isfinite(c.scales[0, page]).all() and (c.scales[0, page] > 0).all()
        for got, want, arith, top in zip(c.values(0, c.streams[0], n), (want_k, want_v),
                                         (2.0 ** -19 * mag + 2.0 ** -145, torch.zeros_like(want_v)),
                                         (448.0, 127.0 if kv == "e4i8" else 448.0)):
            assert torch.isfinite(got).all()
            # half a step (of e4m3, or its subnormals, or int8) at the scale max(amax / top, 2^-126); the arithmetic
            # before it, in f32 down to its subnormals; the quotient's 3 U of up to `top` steps
            amax = want.abs().amax(-1, keepdim=True)
            scale = (amax / top).clamp_min(2.0 ** -126)
            step = 0.5 * scale if top == 127.0 else torch.maximum(want.abs() * 2.0 ** -4, scale * 2.0 ** -10)
            assert not ((got - want).abs() > step * (1 + 2.0 ** -6) + 2 * arith + 2.0 ** -19 * amax).any()


@pytest.mark.parametrize("sections,interleaved,pairs_of", [
    ((24, 20, 20), False, [range(0, 24), range(24, 44), range(44, 64)]),
    ((24, 20, 20), True, [[*range(0, 60, 3), 60, 61, 62, 63], range(1, 60, 3), range(2, 60, 3)]),
    ((62, 1, 1), True, [[0, *range(3, 64)], [1], [2]]),
    ((22, 21, 21), True, [range(0, 64, 3), range(1, 64, 3), range(2, 64, 3)]),
    ((0, 0, 64), False, [[], [], range(0, 64)])])
def test_append_turns_the_pairs_of_an_axis(pkg, sections, interleaved, pairs_of):
    """With a position on one axis alone, the listed pairs turn and the others stay as they are."""
    with Cache(pkg, "f32", [3]) as c:
        gen = torch.Generator(device="cuda").manual_seed(9)
        qkv = torch.randn((1, QKV), device="cuda", generator=gen).expand(3, -1).contiguous()
        q = torch.empty((4, HQ * D), device="cuda")
        slots, pos = i32([c.streams[0]] * 3), i32(range(3))
        for rows, axes, out in ((3, [[5, 0, 0], [0, 5, 0], [0, 0, 5]], q[:3]), (1, [[0]] * 3, q[3:])):
            a = i32(axes)
            c.dec.chunk_append(0, rows, slots.data_ptr(), pos.data_ptr(), a.data_ptr(), sections, interleaved, qkv.data_ptr(),
                               out.data_ptr(), pkg.F32)
            c.dec.sync()
        lo, hi = q.view(4, HQ, 2, 64).unbind(2)
        for axis, pairs in enumerate(pairs_of):
            turned = torch.zeros(64, dtype=torch.bool, device="cuda")
            turned[list(pairs)] = True
            same = ((lo[axis] == lo[3]) & (hi[axis] == hi[3])).all(0)
            assert torch.equal(same, ~turned), axis
