"""Values at the edge of what the chunk operators take: vectors with scale zero, queries that are not finite, moves
between streams that share pages."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_chunk import D, HQ, PT, Cache, check_attend, run_attend, to_i64  # noqa: E402,F401

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
