"""The chunk operators of the paged cache against plain implementations in 64
bits: the append with a rotary position per axis, the attention of a chunk
(causal and draft-tree masks), page copies, token moves, fork and truncate, and
a run of them together."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

D, HQ, HKV, PT = 128, 16, 8, 16
QKV = (HQ + 2 * HKV) * D
THETA, EPS = 1.0e6, 1.0e-6
HALF_BF16, U = 2.0 ** -8, 2.0 ** -24
KINDS = ["f32", "bf16", "fp8", "e4i8"]
NEG = -(1 << 31)


def i32(a):
    return torch.tensor(np.asarray(a, np.int64), dtype=torch.int32, device="cuda")


class Memory:
    def __init__(self, ptr, nbytes):
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (ptr, False), "version": 3}


class Cache:
    """A kv-only decoder with its pool wrapped as a tensor [layers, pages, K|V, head, token, dim]."""

    def __init__(self, pkg, kv, lens=(), layers=1, max_streams=None, spare=4, seed=3, max_context=None):
        rng = np.random.default_rng(seed)
        self.pkg, self.kind, self.layers = pkg, kv, layers
        kv_dtype = {"f32": pkg.F32, "bf16": pkg.BF16, "fp8": pkg.FP8, "e4i8": pkg.E4I8}[kv]
        self.qn = (1.0 + 0.1 * rng.standard_normal((layers, D))).astype(np.float32)
        self.kn = (1.0 + 0.1 * rng.standard_normal((layers, D))).astype(np.float32)
        cfg = dict(n_layers=layers, hidden=256, n_heads=HQ, n_kv_heads=HKV, head_dim=D, intermediate=512, vocab=1000,
                   rope_theta=THETA, rms_norm_eps=EPS)
        pages = sum((n + PT - 1) // PT for n in lens) + spare
        rt = pkg.runtime_config(device=0, kv_dtype=kv_dtype, max_streams=max_streams or max(len(lens), 1),
                                max_context=max_context or max(list(lens) + [PT]), max_pages=pages, max_batch_tokens=64,
                                page_order_seed=5)
        self.dec = pkg.Decoder.kv_only(cfg, rt, self.qn, self.kn)
        info = self.dec.pool_info()
        dtype = {"f32": torch.float32, "bf16": torch.bfloat16}.get(kv, torch.uint8)
        self.n_pages = pages
        assert info["n_pages"] == pages and info["n_layers"] == layers
        raw = torch.as_tensor(Memory(info["pool"], layers * info["layer_bytes"]), device="cuda")
        self.pool = raw.view(dtype).view(layers, pages, 2, HKV, PT, D)
        self.scales = None
        if kv in ("fp8", "e4i8"):
            raw = torch.as_tensor(Memory(info["scales"], layers * info["scales_layer_floats"] * 4), device="cuda")
            self.scales = raw.view(torch.float32).view(layers, pages, 2, HKV, PT)
        self.streams = [self.dec.open() for _ in lens]
        left = list(lens)
        while any(left):                   # grown in turns, so pages of streams interleave
            for j, s in enumerate(self.streams):
                step = min(left[j], 48)
                if step:
                    self.dec.extend(s, step)
                left[j] -= step

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.pool = self.scales = None
        self.dec.close()

    def fill(self, seed=1):
        """Random contents everywhere: every page, every layer."""
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(self.pool.shape, device="cuda", generator=gen)
        if self.scales is None:
            self.pool.copy_(x)
            return
        amax = x.abs().amax(-1, keepdim=True)
        scale = amax / 448.0
        codes = (x / scale).to(torch.float8_e4m3fn).view(torch.uint8)
        if self.kind == "e4i8":
            scale[:, :, 1] = amax[:, :, 1] / 127.0
            codes[:, :, 1] = ((x[:, :, 1] / scale[:, :, 1]).round().clamp(-127, 127) + 128).to(torch.uint8)
        self.pool.copy_(codes)
        self.scales.copy_(scale[..., 0])

    def poison_behind(self, lens):
        """NaN (or NaN codes and scales) in every place of the pool that holds no token."""
        used = torch.zeros((self.n_pages, PT), dtype=torch.bool, device="cuda")
        for s, n in zip(self.streams, lens):
            for k, page in enumerate(self.dec.pages(s)):
                used[int(page), :max(0, min(PT, n - k * PT))] = True
        behind = ~used[None, :, None, None, :, None].expand(self.pool.shape)
        if self.scales is None:
            self.pool[behind] = float("nan")
        else:
            self.pool[behind] = 0x7F
            self.scales[behind[..., 0]] = float("nan")

    def values(self, layer, s, n):
        """K and V of the first n tokens as f64 values, [n, head, dim]."""
        pages = torch.tensor(self.dec.pages(s)[:(n + PT - 1) // PT].astype(np.int64), device="cuda")
        raw = self.pool[layer, pages]
        if self.scales is not None:
            sc = self.scales[layer, pages].double()[..., None]
            k = raw[:, 0].view(torch.float8_e4m3fn).double() * sc[:, 0]
            v = raw[:, 1].double() - 128 if self.kind == "e4i8" else raw[:, 1].view(torch.float8_e4m3fn).double()
            v = v * sc[:, 1]
        else:
            k, v = raw[:, 0].double(), raw[:, 1].double()
        return [t.permute(0, 2, 1, 3).reshape(-1, HKV, D)[:n] for t in (k, v)]


def attend_oracle(q, k, v, seen):
    """q [m, 16, 128], k/v [n, 8, 128], seen [m, n]: (out, sum of p |v|) in f64."""
    out = torch.zeros_like(q)
    mag = torch.zeros_like(q)
    for h in range(HQ):
        logit = (q[:, h] @ k[:, h // 2].T) / math.sqrt(D)
        logit = logit.masked_fill(~seen, -math.inf)
        top = logit.amax(1, keepdim=True)
        e = torch.where(seen, torch.exp(logit - top), torch.zeros_like(logit))
        total = e.sum(1, keepdim=True)
        p = torch.where(total > 0, e / total, torch.zeros_like(e))
        out[:, h], mag[:, h] = p @ v[:, h // 2], p @ v[:, h // 2].abs()
    return out, mag


def attend_tolerance(want, mag):
    """Each probability (times its V scale) is rounded once to bf16: off by 2^-8 of sum p |v| at most; the output once
    more: 2^-8 of itself.  Scores are f32 sums of exact products: |error| < 128 2^-24 sum |q k| / sqrt(128) < 1e-4
    relative in p for |q|, |k| as drawn here, and exp and the f32 sums stay below as much again: 2^-12 in all."""
    return (HALF_BF16 + 2.0 ** -12) * mag + HALF_BF16 * want.abs() + 1e-30


def visible(base, m, bits=None):
    t = torch.arange(base + m, device="cuda")
    if bits is None:
        return t[None] <= base + torch.arange(m, device="cuda")[:, None]
    rows = [[True] * base + [bool(b >> j & 1) for j in range(m)] for b in bits]
    return torch.tensor(rows, device="cuda", dtype=torch.bool).view(m, base + m)


def to_i64(bits):
    return torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64, device="cuda")


def run_attend(cache, chunks, q, starts, masks=None, rows=None, slots=None, lens=None, layer=0, stream=None):
    """chunks [(base, m)]; returns out, which starts out as a pattern."""
    out = torch.full_like(q, -77.0)
    slots = i32(cache.streams[:len(chunks)] if slots is None else slots)
    lens_d = i32([b + m for b, m in chunks] if lens is None else lens)
    starts_d = i32(starts)
    mask = to_i64(masks) if masks is not None else None
    torch.cuda.synchronize()
    cache.dec.chunk_attend(layer, len(chunks), slots.data_ptr(), starts_d.data_ptr(), lens_d.data_ptr(),
                           q.shape[0] if rows is None else rows, mask.data_ptr() if mask is not None else None,
                           q.data_ptr(), out.data_ptr(), stream)
    cache.dec.sync()
    return out


def check_attend(cache, chunks, q, starts, out, masks=None, layer=0):
    touched = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    for j, (base, m) in enumerate(chunks):
        if m == 0:
            continue
        rows = slice(starts[j], starts[j] + m)
        touched[rows] = True
        k, v = cache.values(layer, cache.streams[j], base + m)
        bits = masks[rows] if masks is not None else None
        want, mag = attend_oracle(q[rows].double().view(m, HQ, D), k, v, visible(base, m, bits))
        err = (out[rows].double().view(m, HQ, D) - want).abs()
        over = err > attend_tolerance(want, mag)
        assert not over.any(), (cache.kind, j, base, m, err.max().item(), int(over.sum()))
    assert (out[~touched] == -77.0).all()      # rows of no chunk stay as they were


CHUNKS = {
    "one": [(0, 1)],
    "first_tokens": [(0, 1), (0, 2), (0, 15), (0, 16), (0, 17), (0, 64), (0, 65), (0, 128), (0, 129)],
    "one_new": [(1, 1), (15, 1), (16, 1), (127, 1), (128, 1), (129, 1), (1000, 1)],
    "short": [(511, 5), (120, 9), (0, 3), (2050, 8), (16, 33), (255, 64)],
    "around_a_block": [(0, 63), (64, 64), (1, 65), (127, 127), (128, 128), (129, 129), (300, 257), (0, 385)],
    "ragged": [(700, 3), (3, 300), (0, 0), (1999, 1), (64, 70), (0, 0), (257, 128), (90, 511)],
    "long_context": [(9001, 4)],
    "two_long": [(5003, 77), (4097, 200)],
}


@pytest.mark.parametrize("kv", ["bf16", "fp8", "e4i8"])
@pytest.mark.parametrize("name", list(CHUNKS))
def test_attend_causal(pkg, kv, name):
    chunks = CHUNKS[name]
    lens = [b + m for b, m in chunks]
    gap = 3                                    # rows before the first and behind the last chunk
    starts = [gap + sum(m for _, m in chunks[:j]) for j in range(len(chunks) + 1)]
    with Cache(pkg, kv, lens) as c:
        c.fill()
        c.poison_behind(lens)
        gen = torch.Generator(device="cuda").manual_seed(2)
        q = (1.3 * torch.randn((starts[-1] + gap, HQ * D), device="cuda", generator=gen)).to(torch.bfloat16)
        out = run_attend(c, chunks, q, starts)
        check_attend(c, chunks, q, starts, out)


@pytest.mark.parametrize("kv", ["bf16", "fp8", "e4i8"])
def test_attend_tree_masks(pkg, kv):
    """Random trees, rows that see nothing of the chunk, rows that see nothing at all, bits past the chunk."""
    rng = np.random.default_rng(4)
    chunks = [(0, 5), (600, 8), (0, 64), (1500, 64), (31, 1), (0, 1), (129, 17)]
    masks = []
    for j, (_, m) in enumerate(chunks):
        own = []
        for r in range(m):
            parent = own[int(rng.integers(0, r))] if r else 0
            own.append(parent | 1 << r)
        own[m // 2] = 0                        # an empty row (its stream has no prefix: nothing at all)
        if m > 3:
            own[3] = 1 << (m - 1)              # a later token only
            own[1] |= (1 << 64) - (1 << m)     # bits that name no token of the chunk
        masks += own
    lens = [b + m for b, m in chunks]
    starts = [sum(m for _, m in chunks[:j]) for j in range(len(chunks) + 1)]
    with Cache(pkg, kv, lens) as c:
        c.fill()
        c.poison_behind(lens)
        gen = torch.Generator(device="cuda").manual_seed(2)
        q = (1.3 * torch.randn((starts[-1], HQ * D), device="cuda", generator=gen)).to(torch.bfloat16)
        out = run_attend(c, chunks, q, starts, masks)
        check_attend(c, chunks, q, starts, out, masks)
        assert (out[2] == 0).all() and (out[starts[5]] == 0).all()


@pytest.mark.parametrize("kv", ["bf16", "e4i8"])
def test_attend_extreme_scores(pkg, kv):
    """One key takes all the weight, scores fall from tile to tile or rise with it, and tiny scales."""
    chunks = [(1000, 6), (40, 130)]
    lens = [b + m for b, m in chunks]
    starts = [0, 6, 136]
    with Cache(pkg, kv, lens) as c:
        c.fill()
        gen = torch.Generator(device="cuda").manual_seed(5)
        q = torch.randn((136, HQ * D), device="cuda", generator=gen).to(torch.bfloat16)
        q[:3] *= 30.0                          # scores near +-1000: almost one-hot rows
        q[3] = 0.0                             # a uniform row
        if kv == "bf16":
            for t, f in ((5, 40.0), (500, 80.0), (999, 160.0)):
                page = int(c.dec.pages(c.streams[0])[t // PT])
                c.pool[0, page, 0, :, t % PT] *= f
        else:
            c.scales[:, :, 0] *= torch.logspace(-8, 1, c.n_pages, device="cuda")[None, :, None, None]
            c.scales[:, :, 1] *= 1e-6
        out = run_attend(c, chunks, q, starts)
        # scores reach thousands here, so their f32 rounding reaches the weights: 128 2^-24 sum|q k|/sqrt(128) per row
        for j, (base, m) in enumerate(chunks):
            k, v = c.values(0, c.streams[j], base + m)
            qs = q[starts[j]:starts[j + 1]].double().view(m, HQ, D)
            want, mag = attend_oracle(qs, k, v, visible(base, m))
            prods = torch.einsum("mhd,nhd->mhn", qs.abs(), k.abs().repeat_interleave(2, 1)) / math.sqrt(D)
            ds = (128 * U * prods.amax(-1) + 2.0 ** -12)[..., None]
            tol = attend_tolerance(want, mag) + 2 * ds * mag
            err = (out[starts[j]:starts[j + 1]].double().view(m, HQ, D) - want).abs()
            assert not (err > tol).any(), (j, (err / tol).max().item())


def test_attend_slots_twice_padding_and_layers(pkg):
    """One stream under two entries, padding entries between, the second layer's pool."""
    chunks = [(200, 7), (0, 0), (200, 7), (64, 3)]
    with Cache(pkg, "bf16", [207, 67], layers=2) as c:
        c.fill()
        s = c.streams
        starts = [0, 7, 9, 16, 19]             # the padding entry covers rows 7 and 8
        gen = torch.Generator(device="cuda").manual_seed(2)
        q = torch.randn((21, HQ * D), device="cuda", generator=gen).to(torch.bfloat16)
        q[9:16] = q[:7]
        out = run_attend(c, chunks, q, starts, slots=[s[0], -1, s[0], s[1]], lens=[207, 50, 207, 67], layer=1)
        assert torch.equal(out[:7], out[9:16]) and (out[7:9] == -77).all() and (out[19:] == -77).all()
        for j, rows, n in ((0, slice(0, 7), 207), (1, slice(16, 19), 67)):
            k, v = c.values(1, s[j], n)
            m = rows.stop - rows.start
            want, mag = attend_oracle(q[rows].double().view(m, HQ, D), k, v, visible(n - m, m))
            assert not ((out[rows].double().view(m, HQ, D) - want).abs() > attend_tolerance(want, mag)).any()


@pytest.mark.parametrize("bad", ["slot", "len", "short", "start", "rows", "mask"])
def test_attend_bad_entries_are_reported_and_skipped(pkg, bad):
    chunks = [(100, 4), (50, 4), (30, 4)]
    lens = [104, 54, 34]
    starts = [0, 4, 8, 12]
    masks = None
    with Cache(pkg, "bf16", lens, max_context=112) as c:
        c.fill()
        slots, rows = list(c.streams), 12
        if bad == "slot":
            slots[1] = 99
        elif bad == "len":
            lens[1] = 100000
        elif bad == "short":
            lens[1] = 3                        # fewer tokens than rows
        elif bad == "start":
            starts = [0, 4, 2, 12]
        elif bad == "rows":
            rows = 9
        else:
            starts, masks = [0, 4, 70, 74], [1] * 74
            rows = 74
        gen = torch.Generator(device="cuda").manual_seed(2)
        q = torch.randn((max(rows, 12), HQ * D), device="cuda", generator=gen).to(torch.bfloat16)
        with pytest.raises(pkg.QkvError) as ei:
            run_attend(c, chunks, q, starts, masks=masks, rows=rows, slots=slots, lens=lens)
        assert ei.value.code == 5
        # the handle stays usable, and the other entries' rows are right
        out = torch.full_like(q, -77.0)
        d = [i32(slots), i32(starts), i32(lens)]
        mask = to_i64(masks) if masks else None
        c.dec.chunk_attend(0, 3, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), rows,
                           mask.data_ptr() if masks else None, q.data_ptr(), out.data_ptr())
        torch.cuda.synchronize()
        with pytest.raises(pkg.QkvError):
            c.dec.sync()
        k, v = c.values(0, c.streams[0], 104)
        seen = visible(100, 4, [1] * 4 if masks else None)
        want, mag = attend_oracle(q[:4].double().view(4, HQ, D), k, v, seen)
        assert not ((out[:4].double().view(4, HQ, D) - want).abs() > attend_tolerance(want, mag)).any()
        if bad == "rows":                      # the last entry is the one that does not fit
            assert (out[8:] == -77).all()
        elif bad != "start":
            assert (out[4:8] == -77).all()


def test_attend_refusals(pkg):
    with Cache(pkg, "f32", [20]) as c:
        buf = torch.zeros(4096, dtype=torch.int32, device="cuda")
        a = buf.data_ptr()
        with pytest.raises(pkg.QkvError) as ei:
            c.dec.chunk_attend(0, 1, a, a, a, 1, None, a, a)
        assert ei.value.code == 8
    with Cache(pkg, "bf16", [20]) as c:
        buf = torch.zeros(4096, dtype=torch.int32, device="cuda")
        a = buf.data_ptr()
        for args, code in (((1, 1, a, a, a, 1, None, a, a), 1), ((-1, 1, a, a, a, 1, None, a, a), 1),
                           ((0, -1, a, a, a, 1, None, a, a), 1), ((0, 1, a, a, a, -1, None, a, a), 1),
                           ((0, 1, None, a, a, 1, None, a, a), 1), ((0, 1, a, None, a, 1, None, a, a), 1),
                           ((0, 1, a, a, None, 1, None, a, a), 1), ((0, 1, a, a, a, 1, None, None, a), 1),
                           ((0, 1, a, a, a, 1, None, a, None), 1), ((0, 1025, a, a, a, 1, None, a, a), 3),
                           ((0, 1, a, a, a, (1 << 20) + 1, None, a, a), 3), ((0, 1, a, a, a, 1, None, a + 8, a), 1),
                           ((0, 1, a, a, a, 1, None, a, a + 2), 1)):
            with pytest.raises(pkg.QkvError) as ei:
                c.dec.chunk_attend(*args)
            assert ei.value.code == code, args
        c.dec.chunk_attend(0, 0, None, None, None, 0, None, None, None)
        c.dec.sync()


# ---- append ----

def axis_of_pairs(sections, interleaved):
    if interleaved:
        return [i % 3 if i < 3 * sections[i % 3] else 0 for i in range(64)]
    return [0] * sections[0] + [1] * sections[1] + [2] * sections[2]


def append_oracle(x, w, axes, axis):
    """x [n, heads, 128] f64: (normed and rotated, |u| + |v| of each pair)."""
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    freq = THETA ** (-torch.arange(64, dtype=torch.float64, device="cuda") / 64)
    ang = (axes[torch.tensor(axis, device="cuda")].double().T * freq)[:, None]
    a, b = y[..., :64], y[..., 64:]
    out = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
    return out, (a.abs() + b.abs()).repeat(1, 1, 2)


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("q_bf16", [False, True])
@pytest.mark.parametrize("sections,interleaved", [((24, 20, 20), True), ((24, 20, 20), False), ((64, 0, 0), False),
                                                  ((0, 64, 0), False), ((22, 21, 21), True)])
def test_append(pkg, kv, q_bf16, sections, interleaved):
    lens = [1, 70, 33]
    with Cache(pkg, kv, lens, layers=2) as c:
        c.fill()
        before = c.pool.clone()
        sc_before = c.scales.clone() if c.scales is not None else None
        rng = np.random.default_rng(6)
        rows = [(j, t) for j, n in enumerate(lens) for t in range(n) if n < 40 or t % 3]
        rng.shuffle(rows)
        n = len(rows) + 2                      # the first and the last row are padding
        slots = [-1] + [c.streams[j] for j, _ in rows] + [-1]
        pos = [0] + [t for _, t in rows] + [0]
        axes = rng.integers(-5000, 5000, (3, n))
        axes[:, 3] = (2 ** 31 - 1, -2 ** 31, 123456789)
        axes[:, 4] = (0, 0, 0)
        axes[:, 5] = (1000003, 250000, 99999)
        axes = torch.tensor(axes, dtype=torch.int32, device="cuda")
        gen = torch.Generator(device="cuda").manual_seed(7)
        qkv = torch.randn((n, QKV), device="cuda", generator=gen)
        qkv[4] *= 1e-3
        qkv[5] *= 300.0
        qkv[6] = 0.0
        q_out = torch.full((n, HQ * D), -77.0, device="cuda", dtype=torch.bfloat16 if q_bf16 else torch.float32)
        d_slots, d_pos = i32(slots), i32(pos)
        c.dec.chunk_append(1, n, d_slots.data_ptr(), d_pos.data_ptr(), axes.data_ptr(), sections, interleaved,
                           qkv.data_ptr(), q_out.data_ptr(), pkg.BF16 if q_bf16 else pkg.F32)
        c.dec.sync()
        assert (q_out[0] == -77).all() and (q_out[-1] == -77).all()
        axis = axis_of_pairs(sections, interleaved)
        x = qkv.double()
        qn, kn = [torch.tensor(w[1], device="cuda").double() for w in (c.qn, c.kn)]
        want_q, mag_q = append_oracle(x[:, :2048].view(n, HQ, D), qn, axes, axis)
        want_k, mag_k = append_oracle(x[:, 2048:2048 + 1024].view(n, HKV, D), kn, axes, axis)
        want_v = x[:, 2048 + 1024:].view(n, HKV, D)
        # Norm: a sum of 128 squares over 8 serial and 4 pairwise steps (12 roundings, halved by the root), root,
        # quotient and two products: under 12 U.  Angle: the fraction of a turn rounded to float (pi U), sincospi's
        # 2 ulp: under 8 U.  Rotation: two products and a sum, 3 U.  All relative to |u| + |v|: 23 U < 2^-19.
        rot = 2.0 ** -19
        got = q_out.double().view(n, HQ, D)[1:-1]
        tol = rot * mag_q[1:-1] + (HALF_BF16 * want_q[1:-1].abs() if q_bf16 else 0) + 1e-30
        assert not ((got - want_q[1:-1]).abs() > tol).any()

        page_of = {j: c.dec.pages(s) for j, s in enumerate(c.streams)}
        pg = torch.tensor([int(page_of[j][t // PT]) for j, t in rows], device="cuda")
        tk = torch.tensor([t % PT for _, t in rows], device="cuda")
        for kv_half, want, mag in ((0, want_k[1:-1], mag_k[1:-1]), (1, want_v[1:-1], None)):
            arith = rot * mag if mag is not None else torch.zeros_like(want)
            raw = c.pool[1, pg, kv_half, :, tk]
            if kv == "f32":
                assert not ((raw.double() - want).abs() > arith + 1e-30).any()
            elif kv == "bf16":
                assert not ((raw.double() - want).abs() > arith + HALF_BF16 * want.abs() + 1e-30).any()
            else:
                i8 = kv == "e4i8" and kv_half == 1
                top = 127.0 if i8 else 448.0
                scale = c.scales[1, pg, kv_half, :, tk].double()
                amax = want.abs().amax(-1)
                live = amax > 0
                assert not ((scale - amax / top).abs()[live] > (2 * U * amax + arith.amax(-1))[live] / top).any()
                assert (scale[~live] == 1).all()
                val = (raw.double() - 128 if i8 else raw.view(torch.float8_e4m3fn).double()) * scale[..., None]
                # half a step: int8 half the scale; e4m3 2^-4 of the value, or half its subnormal step 2^-9 of the
                # scale; the quotient x / scale is off by 3 U of up to `top` steps, which moves a tie by as much
                step = scale[..., None] * 0.5 if i8 else torch.maximum(want.abs() * 2.0 ** -4, scale[..., None] * 2.0 ** -10)
                assert not ((val - want).abs() > step * (1 + 2.0 ** -6) + 2 * arith + 2.0 ** -19 * amax[..., None]).any()
            if kv_half == 1 and kv in ("f32", "bf16"):     # v is stored as it comes, rounded once
                assert torch.equal(raw, want.float().to(raw.dtype))
        # nothing else of the pool has moved
        keep = torch.ones((c.n_pages, PT), dtype=torch.bool, device="cuda")
        keep[pg, tk] = False
        same = keep[:, None, None, :, None].expand(c.pool.shape[1:])
        view = (lambda t: t.view(torch.int16)) if kv == "bf16" else (lambda t: t)
        assert torch.equal(view(c.pool)[0], view(before)[0]) and torch.equal(view(c.pool)[1][same], view(before)[1][same])
        if sc_before is not None:
            assert torch.equal(c.scales[0], sc_before[0]) and torch.equal(c.scales[1][same[..., 0]], sc_before[1][same[..., 0]])


@pytest.mark.parametrize("kv", KINDS)
def test_append_with_equal_axes_is_the_plain_append(pkg, kv):
    """Positions equal on all axes and to the cache position: what kv_append stores, to its last bits."""
    lens = [300]
    with Cache(pkg, kv, lens, layers=2) as c:
        n = 300
        gen = torch.Generator(device="cuda").manual_seed(7)
        qkv = torch.randn((n, QKV), device="cuda", generator=gen)
        slots, pos = i32([c.streams[0]] * n), i32(range(n))
        axes = torch.stack([pos] * 3).contiguous()
        q = [torch.empty((n, HQ * D), device="cuda") for _ in range(2)]
        # the two layers have their own norm weights: use layer 0 for both, and compare with a copy
        c.dec.kv_append(0, n, slots.data_ptr(), pos.data_ptr(), qkv.data_ptr(), q[0].data_ptr())
        torch.cuda.synchronize()
        k0, v0 = [t.clone() for t in c.values(0, c.streams[0], n)]
        c.pool.zero_()
        c.dec.chunk_append(0, n, slots.data_ptr(), pos.data_ptr(), axes.data_ptr(), (24, 20, 20), True, qkv.data_ptr(),
                           q[1].data_ptr(), pkg.F32)
        c.dec.sync()
        k1, v1 = c.values(0, c.streams[0], n)
        # both are within 2^-19 (|u| + |v|) of the exact values, |u| + |v| <= sqrt(2) max |head|
        assert (q[0] - q[1]).abs().max() <= 2.0 ** -17 * q[0].abs().max()
        assert torch.equal(v0, v1)
        step = {"f32": 2.0 ** -17, "bf16": 2 * HALF_BF16, "fp8": 2.0 ** -3, "e4i8": 2.0 ** -3}[kv]
        assert (k0 - k1).abs().max() <= step * k0.abs().max()


def test_append_bad_rows_and_refusals(pkg):
    with Cache(pkg, "bf16", [40, 20]) as c:
        c.fill()
        n = 4
        gen = torch.Generator(device="cuda").manual_seed(7)
        qkv = torch.randn((n, QKV), device="cuda", generator=gen)
        axes = torch.zeros((3, n), dtype=torch.int32, device="cuda")
        for slots, pos in (([0, 7, 1, 0], [0, 0, 0, 1]), ([0, NEG, 1, 0], [0, 0, 0, 1]),
                           ([0, 0, 1, 0], [0, 2 ** 31 - 1, 0, 1]), ([0, 0, 1, 0], [0, -1, 0, 1]),
                           ([0, 1, 1, 0], [0, 32, 0, 1])):      # a page the stream does not own
            q = torch.full((n, HQ * D), -77.0, device="cuda")
            before = c.pool.clone()
            d = [i32([c.streams[s] if 0 <= s < 2 else s for s in slots]), i32(pos)]
            c.dec.chunk_append(0, n, d[0].data_ptr(), d[1].data_ptr(), axes.data_ptr(), (64, 0, 0), False, qkv.data_ptr(),
                               q.data_ptr(), pkg.F32)
            torch.cuda.synchronize()
            with pytest.raises(pkg.QkvError) as ei:
                c.dec.sync()
            assert ei.value.code == 5
            assert (q[1] == -77).all() and (q[[0, 2, 3]] != -77).any(1).all()
            assert (c.pool != before).any(-1).sum() <= 3 * 2 * HKV
        a = qkv.data_ptr()
        for args, code in (((1, 1, a, a, a, (64, 0, 0), 0, a, a, 0), 1), ((0, -1, a, a, a, (64, 0, 0), 0, a, a, 0), 1),
                           ((0, 1, None, a, a, (64, 0, 0), 0, a, a, 0), 1), ((0, 1, a, a, None, (64, 0, 0), 0, a, a, 0), 1),
                           ((0, 1, a, a, a, (24, 20, 21), 0, a, a, 0), 1), ((0, 1, a, a, a, (70, -6, 0), 0, a, a, 0), 1),
                           ((0, 1, a, a, a, (20, 22, 22), 1, a, a, 0), 1), ((0, 1, a, a, a, (64, 0, 0), 0, a, a, 2), 1),
                           ((0, 1, a, a, a, (64, 0, 0), 0, a + 4, a, 0), 1), ((0, 1, a, a, a, (64, 0, 0), 0, a, a + 8, 0), 1)):
            with pytest.raises(pkg.QkvError) as ei:
                c.dec.chunk_append(*args)
            assert ei.value.code == code, args
        with pytest.raises(ValueError):
            c.dec.chunk_append(0, 1, a, a, a, (64, 0), 0, a, a, 0)
        c.dec.chunk_append(0, 0, None, None, None, (64, 0, 0), 0, None, None, 0)
        c.dec.sync()


# ---- copies and moves ----

def raw(t):
    return t.view(torch.int16) if t.dtype == torch.bfloat16 else t


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("n", [1, 5, 40])
def test_pages_copy(pkg, kv, n):
    with Cache(pkg, kv, layers=3, spare=2 * n + 3) as c:
        c.fill()
        order = np.random.default_rng(n).permutation(2 * n + 3)
        src, dst = order[:n], order[n:2 * n]
        want = c.pool.clone()
        want[:, dst] = want[:, src]
        sc = c.scales.clone() if c.scales is not None else None
        if sc is not None:
            sc[:, dst] = sc[:, src]
        d = [i32(src), i32(dst)]
        c.dec.pages_copy(n, d[0].data_ptr(), d[1].data_ptr())
        c.dec.sync()
        assert torch.equal(raw(c.pool), raw(want)) and (sc is None or torch.equal(c.scales, sc))


def test_pages_copy_bad_pages(pkg):
    with Cache(pkg, "bf16", layers=2, spare=8) as c:
        c.fill()
        want = c.pool.clone()
        want[:, 5] = want[:, 2]
        for bad in ([-1, 1], [8, 1], [1, 8], [1, NEG]):
            d = [i32([bad[0], 2]), i32([bad[1], 5])]
            c.dec.pages_copy(2, d[0].data_ptr(), d[1].data_ptr())
            torch.cuda.synchronize()
            with pytest.raises(pkg.QkvError) as ei:
                c.dec.sync()
            assert ei.value.code == 5 and torch.equal(raw(c.pool), raw(want))
        for args in ((-1, 1, 1), (1, None, 1), (1, 1, None)):
            with pytest.raises(pkg.QkvError) as ei:
                c.dec.pages_copy(*args)
            assert ei.value.code == 1
        c.dec.pages_copy(0, None, None)
        c.dec.sync()


def run_move(c, groups, extra=0):
    """groups [(src slot, src base, dst slot, dst base, keep)]"""
    starts = [sum(len(g[4]) for g in groups[:j]) for j in range(len(groups) + 1)]
    d = [i32([g[k] for g in groups]) for k in range(4)] + [i32(starts), i32([t for g in groups for t in g[4]] + [0])]
    p = [t.data_ptr() for t in d]
    c.dec.tokens_move(len(groups), *p[:5], starts[-1] + extra, p[5])
    c.dec.sync()


@pytest.mark.parametrize("kv", KINDS)
def test_tokens_move(pkg, kv):
    """In place (the accepted path closes up), to another stream, more tokens than one batch, empty and padding."""
    lens = [60, 60, 90, 90, 20]
    with Cache(pkg, kv, lens, layers=3) as c:
        c.fill()
        s = c.streams
        groups = [(s[0], 37, s[0], 37, [0, 2, 3, 9, 10, 11, 20]), (s[1], 40, s[1], 30, list(range(20))),
                  (s[2], 5, s[3], 0, list(range(0, 85, 2))), (s[4], 3, s[4], 3, []), (-1, 0, s[4], 0, [1, 2])]
        want = {(j, layer): [t.clone() for t in c.values(layer, s[j], n)] for j, n in enumerate(lens) for layer in range(3)}
        for a, ab, b, bb, keep in groups:
            if a < 0:
                continue
            for layer in range(3):
                src, dst = want[(s.index(a), layer)], want[(s.index(b), layer)]
                for x, y in zip(src, dst):
                    moved = x[[ab + t for t in keep]].clone()
                    y[bb:bb + len(keep)] = moved
        run_move(c, groups)
        for (j, layer), (k, v) in want.items():
            got = c.values(layer, s[j], lens[j])
            assert torch.equal(got[0], k) and torch.equal(got[1], v), (j, layer)


def test_tokens_move_bad_groups(pkg):
    with Cache(pkg, "bf16", [64, 64], layers=2, max_context=96) as c:
        c.fill()
        a, b = c.streams
        before = c.pool.clone()
        for g in ((a, 10, a, 11, [0, 1]), (a, 10, a, 5, [1, 1]), (a, 10, a, 5, [2, 1]), (a, 10, b, 5, [-1, 3]),
                  (a, 60, b, 0, [0, 4]), (a, 0, b, 63, [0, 1]), (a, -1, b, 0, [1, 2]), (a, 0, b, -1, [1, 2]),
                  (9, 0, b, 0, [1]), (a, 0, 9, 0, [1]), (a, 2 ** 31 - 1, b, 0, [1, 2]), (a, 0, b, 2 ** 31 - 1, [1, 2]),
                  (a, 0, b, 0, [1, 2 ** 31 - 1])):
            with pytest.raises(pkg.QkvError) as ei:
                run_move(c, [g])
            assert ei.value.code == 5
            assert torch.equal(raw(c.pool), raw(before)), g
        x = i32([0, 9, 0])
        p = x.data_ptr()
        for args in ((-1, p, p, p, p, p, 1, p), (1, p, p, p, p, p, -1, p), (1, None, p, p, p, p, 1, p),
                     (1, p, p, p, p, p, 1, None)):
            with pytest.raises(pkg.QkvError) as ei:
                c.dec.tokens_move(*args)
            assert ei.value.code == 1
        with pytest.raises(pkg.QkvError) as ei:
            c.dec.tokens_move(65536, p, p, p, p, p, 1, p)
        assert ei.value.code == 3
        c.dec.tokens_move(0, None, None, None, None, None, 0, None)
        c.dec.sync()


# ---- streams ----

@pytest.mark.parametrize("kv", KINDS)
def test_fork_and_truncate_copy_contents(pkg, kv):
    with Cache(pkg, kv, [75], layers=2, max_streams=4, spare=6, max_context=128) as c:
        c.fill()
        dec, a = c.dec, c.streams[0]
        base = [t.clone() for t in c.values(1, a, 75)]

        def same(s, n):
            return all(torch.equal(x, y[:n]) for x, y in zip(c.values(1, s, n), base))

        b = dec.fork(a, 75)
        assert same(b, 75) and list(dec.pages(b)[:4]) == list(dec.pages(a)[:4]) and dec.pages(b)[4] != dec.pages(a)[4]
        d = dec.fork(b, 48)
        dec.sync()
        assert same(d, 48) and dec.pool_stats() == (5, 11)
        dec.truncate(b, 40)                    # inside a page that a and d share
        dec.sync()
        assert same(b, 40) and dec.pages(b)[2] not in set(dec.pages(a)) | set(dec.pages(d))
        c.pool[:, int(dec.pages(b)[2])] = 0    # b's own page: the others keep theirs
        assert same(a, 75) and same(d, 48)
        before = {s: dec.length(s) for s in (a, b, d)}
        dec.compact()
        assert {s: dec.length(s) for s in before} == before and same(a, 75) and same(d, 48)
        table = torch.as_tensor(Memory(dec.pool_info()["page_table"], 4 * 8 * 4), device="cuda").view(torch.int32).view(4, 8)
        for s in before:
            row = table[s].tolist()
            pages = dec.pages(s).tolist()
            assert row == pages + [-1] * (8 - len(pages))
        dec.close_stream(a)
        assert same(d, 48)
        with pytest.raises(pkg.QkvError) as ei:
            dec.fork(a, 0)
        assert ei.value.code == 1
        with pytest.raises(pkg.QkvError) as ei:
            dec.truncate(d, 49)
        assert ei.value.code == 1


def test_fork_and_truncate_refuse_a_captured_stream(pkg):
    with Cache(pkg, "bf16", [20], max_streams=2) as c:
        st = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        x = torch.zeros(4, device="cuda")
        codes = []
        with torch.cuda.graph(g, stream=st):
            x += 1
            for call in (lambda: c.dec.fork(c.streams[0], 20, st.cuda_stream),
                         lambda: c.dec.truncate(c.streams[0], 3, st.cuda_stream)):
                try:
                    call()
                except pkg.QkvError as e:
                    codes.append(e.code)
        assert codes == [8, 8] and c.dec.length(c.streams[0]) == 20
        c.dec.sync()


def test_forked_stream_decodes_as_the_original(pkg, synth, tiny_files):
    """Model level: a fork continues greedily as its source does, and a truncated stream repeats its steps."""
    cfg, files = tiny_files
    path = files[("bf16", "one_plus")]
    rng = np.random.default_rng(3)
    x, _ = synth.prompt_rows(synth.read_gguf(path)["text.token_embd.weight"], 37, rng, audio_rows=20, audio_start=4)
    rt = pkg.runtime_config(device=0, weight_dtype=pkg.BF16, kv_dtype=pkg.BF16, max_streams=3, max_context=96)
    with pkg.Decoder.from_gguf(path, rt) as dec:
        a = dec.open()
        first = dec.prefill([a], [x])[0]
        b = dec.fork(a, 37)
        ids_a = [int(dec.decode_step([a])[0]) for _ in range(6)]
        ids_b = [int(dec.decode_step([b])[0]) for _ in range(6)]
        assert ids_a == ids_b
        dec.truncate(a, 37)
        with pytest.raises(pkg.QkvError):
            dec.decode_step([a])               # no id to go on from
        again = [int(dec.decode_step([a], in_ids=[first])[0])] + [int(dec.decode_step([a])[0]) for _ in range(5)]
        assert again == ids_a


def test_draft_trees_of_forked_streams_together(pkg):
    """The operators as they are used: a shared prompt, forks, draft trees appended and attended to, the accepted path
    kept and the rest given back, a next chunk; every cache and output against a list of tokens kept aside."""
    layers, prompt, draft = 2, 83, 9
    rng = np.random.default_rng(12)
    with Cache(pkg, "bf16", [prompt], layers=layers, max_streams=4, spare=24, max_context=160) as c:
        dec = c.dec
        gen = torch.Generator(device="cuda").manual_seed(13)
        st = torch.cuda.Stream()
        sections = (24, 20, 20)

        def append_attend(streams, bases, depths, masks):
            """One chunk of each stream through every layer; returns q, out per layer."""
            m = [len(d) for d in depths]
            n = sum(m)
            starts = [sum(m[:j]) for j in range(len(m) + 1)]
            pos = [b + t for b, k in zip(bases, m) for t in range(k)]
            rot = [b + t for b, d in zip(bases, depths) for t in d]
            d = dict(row_slots=i32([s for s, k in zip(streams, m) for _ in range(k)]), pos=i32(pos),
                     axes=i32([rot] * 3), slots=i32(streams), starts=i32(starts),
                     lens=i32([b + k for b, k in zip(bases, m)]), mask=to_i64(masks) if masks else None)
            res = []
            for layer in range(layers):
                qkv = torch.randn((n, QKV), device="cuda", generator=gen)
                q = torch.empty((n, HQ * D), device="cuda", dtype=torch.bfloat16)
                out = torch.empty_like(q)
                st.wait_stream(torch.cuda.current_stream())
                dec.chunk_append(layer, n, d["row_slots"].data_ptr(), d["pos"].data_ptr(), d["axes"].data_ptr(), sections,
                                 True, qkv.data_ptr(), q.data_ptr(), pkg.BF16, st.cuda_stream)
                dec.chunk_attend(layer, len(m), d["slots"].data_ptr(), d["starts"].data_ptr(), d["lens"].data_ptr(), n,
                                 d["mask"].data_ptr() if masks else None, q.data_ptr(), out.data_ptr(), st.cuda_stream)
                torch.cuda.current_stream().wait_stream(st)
                res.append((qkv, q, out))
            dec.sync()
            return starts, res

        def rotated_k(qkv, layer, rot):
            n = qkv.shape[0]
            axes = torch.tensor([rot] * 3, device="cuda")
            k, _ = append_oracle(qkv[:, 2048:2048 + 1024].double().view(n, HKV, D), torch.tensor(c.kn[layer], device="cuda").double(),
                                 axes, [0] * 64)
            return k

        # the prompt, in two pieces
        a = c.streams[0]
        cache = {}
        dec.truncate(a, 0, st.cuda_stream)
        done = 0
        for piece in (50, prompt - 50):
            dec.extend(a, piece)
            starts, res = append_attend([a], [done], [list(range(piece))], None)
            for layer, (qkv, q, out) in enumerate(res):
                k, v = rotated_k(qkv, layer, [done + t for t in range(piece)]), qkv[:, 2048 + 1024:].double().view(-1, HKV, D)
                old = cache.get((a, layer))
                cache[(a, layer)] = (k, v) if old is None else tuple(torch.cat([x, y]) for x, y in zip(old, (k, v)))
            done += piece
        streams = [a, dec.fork(a, prompt, st.cuda_stream), dec.fork(a, prompt - 7, st.cuda_stream)]
        lens = [prompt, prompt, prompt - 7]
        for s, n in zip(streams[1:], lens[1:]):
            for layer in range(layers):
                cache[(s, layer)] = tuple(t[:n] for t in cache[(a, layer)])
        for _ in range(3):
            trees, depths = [], []
            for _ in streams:
                bits, depth = [], []
                for r in range(draft):
                    p = int(rng.integers(-1, r)) if r else -1
                    bits.append((bits[p] if p >= 0 else 0) | 1 << r)
                    depth.append(depth[p] + 1 if p >= 0 else 0)
                trees.append(bits)
                depths.append(depth)
            for s in streams:
                dec.extend(s, draft)
            starts, res = append_attend(streams, lens, depths, [b for t in trees for b in t])
            keeps = []
            for j, s in enumerate(streams):
                leaf = int(rng.integers(0, draft))
                keep = [t for t in range(draft) if trees[j][leaf] >> t & 1]
                keeps.append(keep)
                for layer, (qkv, q, out) in enumerate(res):
                    rows = slice(starts[j], starts[j] + draft)
                    k, v = rotated_k(qkv[rows], layer, [lens[j] + t for t in depths[j]]), qkv[rows, 2048 + 1024:].double().view(-1, HKV, D)
                    # the stored cache is bf16 of these: the attention is held to the cache as stored
                    got_k, got_v = c.values(layer, s, lens[j] + draft)
                    all_k, all_v = [torch.cat([x, y]) for x, y in zip(cache[(s, layer)], (k, v))]
                    bound = HALF_BF16 * all_k.abs() + 2.0 ** -17 * all_k.abs().max()
                    assert not ((got_k - all_k).abs() > bound).any()
                    assert not ((got_v - all_v).abs() > HALF_BF16 * all_v.abs()).any()
                    want, mag = attend_oracle(q[rows].double().view(draft, HQ, D), got_k, got_v,
                                              visible(lens[j], draft, trees[j]))
                    assert not ((out[rows].double().view(draft, HQ, D) - want).abs() > attend_tolerance(want, mag)).any()
                    cache[(s, layer)] = tuple(torch.cat([x, y[keep]]) for x, y in zip(cache[(s, layer)], (k, v)))
            counts = [len(k) for k in keeps]
            d = [i32(streams), i32(lens), i32([sum(counts[:j]) for j in range(len(counts) + 1)]),
                 i32([t for k in keeps for t in k])]
            torch.cuda.synchronize()
            p = [t.data_ptr() for t in d]
            dec.tokens_move(len(streams), p[0], p[1], p[0], p[1], p[2], sum(counts), p[3], st.cuda_stream)
            for j, s in enumerate(streams):
                lens[j] += counts[j]
                dec.truncate(s, lens[j], st.cuda_stream)
            dec.sync()
        dec.compact()
        for j, s in enumerate(streams):
            for layer in range(layers):
                got_k, got_v = c.values(layer, s, lens[j])
                k, v = cache[(s, layer)]
                assert not ((got_k - k).abs() > HALF_BF16 * k.abs() + 2.0 ** -17 * k.abs().max()).any()
                assert torch.equal(got_v.float(), v.float().to(torch.bfloat16).float())


def test_chunk_calls_in_a_captured_graph(pkg):
    """A captured append + attend serves other slots, lengths and a smaller batch on replay."""
    lens_a, lens_b = [300, 45], [290, 130]
    with Cache(pkg, "bf16", [300, 130], max_context=320) as c:
        c.fill()
        rows = 12
        gen = torch.Generator(device="cuda").manual_seed(3)
        qkv = torch.randn((rows, QKV), device="cuda", generator=gen)
        q = torch.zeros((rows, HQ * D), device="cuda", dtype=torch.bfloat16)
        out = torch.zeros_like(q)
        row_slots, pos, axes = i32([-1] * rows), i32([0] * rows), i32([[0] * rows] * 3)
        slots, starts, lens = i32([-1, -1]), i32([0, 0, 0]), i32([0, 0])
        st = torch.cuda.Stream()
        torch.cuda.synchronize()

        def call():
            c.dec.chunk_append(0, rows, row_slots.data_ptr(), pos.data_ptr(), axes.data_ptr(), (24, 20, 20), False,
                               qkv.data_ptr(), q.data_ptr(), pkg.BF16, st.cuda_stream)
            c.dec.chunk_attend(0, 2, slots.data_ptr(), starts.data_ptr(), lens.data_ptr(), rows, None, q.data_ptr(),
                               out.data_ptr(), st.cuda_stream)

        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            call()
        for ln, m in ((lens_a, (5, 7)), (lens_b, (9, 3)), (lens_b, (1, 0))):
            chunk_rows = [(c.streams[j], ln[j] - m[j] + t) for j in range(2) for t in range(m[j])]
            pad = rows - len(chunk_rows)
            row_slots.copy_(i32([s for s, _ in chunk_rows] + [-1] * pad))
            pos.copy_(i32([t for _, t in chunk_rows] + [0] * pad))
            axes.copy_(i32([[t for _, t in chunk_rows] + [0] * pad] * 3))
            slots.copy_(i32([c.streams[0], c.streams[1] if m[1] else -1]))
            starts.copy_(i32([0, m[0], m[0] + m[1]]))
            lens.copy_(i32(ln))
            out.fill_(-77.0)
            torch.cuda.synchronize()
            g.replay()
            c.dec.sync()
            chunks = [(ln[j] - m[j], m[j]) for j in range(2)]
            check_attend(c, chunks, q, [0, m[0]], out)


# ---- many entries, wide ranges, large pools ----

def check_entry(c, stream, length, rows, q, out, seen, extra=0.0):
    m = rows.stop - rows.start
    k, v = c.values(0, stream, length)
    want, mag = attend_oracle(q[rows].double().view(m, HQ, D), k, v, seen)
    err = (out[rows].double().view(m, HQ, D) - want).abs()
    over = err > attend_tolerance(want, mag) + extra * mag
    assert not over.any(), (c.kind, stream, length, m, err.max().item(), int(over.sum()))


@pytest.mark.parametrize("kv", ["bf16", "fp8", "e4i8"])
@pytest.mark.parametrize("n,bad", [(32, -1), (33, -1), (200, 77), (1024, -1)])
def test_attend_many_entries(pkg, kv, n, bad):
    """Entries by the hundred: padding between them, empty chunks, prefixes of a stream, a bad one; twice, the same bits."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(1, 400, 24)]
    sizes = [0, 1, 1, 2, 5, 9, 17, 40] + ([70, 130] if n <= 200 else [])
    slots, starts, ends, chunks = [], [0], [], []
    for i in range(n):
        j = int(rng.integers(0, len(lens)))
        m = min(int(rng.choice(sizes)), lens[j])
        end = int(rng.integers(max(m, 1), lens[j] + 1))
        pad = rng.random() < 0.1
        slots.append(-1 if pad else j)
        chunks.append(None if pad or i == bad else (j, end, m))
        ends.append(end)
        starts.append(starts[-1] + m)
    with Cache(pkg, kv, lens) as c:
        c.fill()
        c.poison_behind(lens)
        gen = torch.Generator(device="cuda").manual_seed(2)
        q = (1.3 * torch.randn((starts[-1] + 2, HQ * D), device="cuda", generator=gen)).to(torch.bfloat16)
        ids = i32([999 if i == bad else (-1 if j < 0 else c.streams[j]) for i, j in enumerate(slots)])
        d_starts, d_lens = i32(starts), i32(ends)
        side = torch.cuda.Stream()
        outs = [torch.full_like(q, -77.0) for _ in range(2)]
        torch.cuda.synchronize()
        for out in outs:
            c.dec.chunk_attend(0, n, ids.data_ptr(), d_starts.data_ptr(), d_lens.data_ptr(), q.shape[0], None, q.data_ptr(),
                               out.data_ptr(), side.cuda_stream)
        torch.cuda.synchronize()
        if bad >= 0:
            with pytest.raises(pkg.QkvError) as ei:
                c.dec.sync()
            assert ei.value.code == 5
        else:
            c.dec.sync()
        assert torch.equal(outs[0], outs[1])
        for i, chunk in enumerate(chunks):
            rows = slice(starts[i], starts[i + 1])
            if chunk is None:
                assert (outs[0][rows] == -77).all()
            elif chunk[2]:
                j, end, m = chunk
                check_entry(c, c.streams[j], end, rows, q, outs[0], visible(end - m, m))
        assert (outs[0][starts[-1]:] == -77).all()


def profile(name, n):
    """Size of token t's key along a direction: the scores, in powers of two, are about 16 times as large."""
    t = np.arange(n)
    return {"rising": 80.0 * t / n - 40.0, "falling": 40.0 - 80.0 * t / n, "low": -30.0 + 0.1 * np.sin(t),
            "high": 45.0 + 0.1 * np.sin(t), "steps": np.array([-60.0, -20.0, 20.0, 0.0, 60.0, -5.0])[(t + 64) // 128 % 6],
            "spike": np.where(t == n // 2, 50.0, 0.01 * np.cos(t)), "first": np.where(t == 0, 50.0, -0.3)}[name]


@pytest.mark.parametrize("kv", ["bf16", "fp8", "e4i8"])
@pytest.mark.parametrize("name", ["rising", "falling", "low", "high", "steps", "spike", "first"])
def test_attend_score_profiles(pkg, kv, name):
    """Scores that run through hundreds of powers of two along the keys, for every number of rows at a time."""
    chunks = [(660, 5), (663, 14), (650, 40), (600, 130), (0, 200), (3, 12)]
    lens = [b + m for b, m in chunks]
    starts = [sum(m for _, m in chunks[:j]) for j in range(len(chunks) + 1)]
    with Cache(pkg, kv, lens) as c:
        c.fill()
        gen = torch.Generator(device="cuda").manual_seed(8)
        u = torch.randint(0, 2, (HKV, D), device="cuda", generator=gen).float() * 2 - 1
        for s, n in zip(c.streams, lens):
            coef = torch.tensor(profile(name, n), dtype=torch.float32, device="cuda")
            t = torch.arange(n, device="cuda")
            page = torch.tensor(c.dec.pages(s).astype(np.int64), device="cuda")[t // PT]
            if kv == "bf16":
                c.pool[0, page, 0, :, t % PT] = (coef[:, None, None] * u).to(torch.bfloat16)
            else:
                code = torch.where(coef[:, None, None] * u >= 0, 0x38, 0xB8).to(torch.uint8)   # +-1
                c.pool[0, page, 0, :, t % PT] = code
                c.scales[0, page, 0, :, t % PT] = coef.abs()[:, None].clamp_min(1e-30).expand(-1, HKV).contiguous()
        c.poison_behind(lens)
        size = torch.ones((starts[-1], 1, 1), device="cuda")
        size[1::4] = -1.0                     # these rows go through the profile upside down
        size[2::4] = 0.01
        q = size * u.repeat_interleave(2, 0) + 0.02 * torch.randn((starts[-1], HQ, D), device="cuda", generator=gen)
        q = q.reshape(-1, HQ * D).to(torch.bfloat16)
        out = run_attend(c, chunks, q, starts)
        # the f32 rounding of scores in the hundreds reaches the weights: 128 2^-24 sum |q k| / sqrt(128) each way
        for j, (base, m) in enumerate(chunks):
            k, _ = c.values(0, c.streams[j], base + m)
            rows = slice(starts[j], starts[j + 1])
            qs = q[rows].double().view(m, HQ, D)
            top = (torch.einsum("mhd,nhd->mhn", qs.abs(), k.abs().repeat_interleave(2, 1)) / math.sqrt(D)).max().item()
            check_entry(c, c.streams[j], base + m, rows, q, out, visible(base, m), 2 * (128 * U * top + 2.0 ** -12))


def test_attend_mask_alignment_and_large_values(pkg):
    with Cache(pkg, "bf16", [300, 300]) as c:
        c.fill()
        buf = torch.zeros(4096, dtype=torch.int64, device="cuda")
        a = buf.data_ptr()
        with pytest.raises(pkg.QkvError) as ei:
            c.dec.chunk_attend(0, 1, a, a, a, 1, a + 4, a, a)
        assert ei.value.code == 1
        c.pool[:, :, 1] *= 2.0 ** 61           # exact; largest magnitude below 2^64
        gen = torch.Generator(device="cuda").manual_seed(2)
        q = torch.randn((80, HQ * D), device="cuda", generator=gen).to(torch.bfloat16)
        chunks, starts = [(290, 10), (230, 70)], [0, 10, 80]
        check_attend(c, chunks, q, starts, run_attend(c, chunks, q, starts))


def test_attend_refuses_more_work_than_it_counts(pkg):
    """2^20 rows where each could see 2^21 tokens: past 2^31 units of work; a few rows there are served."""
    with Cache(pkg, "bf16", [300], max_context=1 << 21) as c:
        c.fill()
        gen = torch.Generator(device="cuda").manual_seed(2)
        q = torch.randn((300, HQ * D), device="cuda", generator=gen).to(torch.bfloat16)
        with pytest.raises(pkg.QkvError) as ei:
            run_attend(c, [(0, 300)], q, [0, 300], rows=1 << 20)
        assert ei.value.code == 3
        check_attend(c, [(0, 300)], q, [0, 300], run_attend(c, [(0, 300)], q, [0, 300]))


def test_attend_reports_missing_pages(pkg):
    """A length that reaches pages the stream does not have: reported; the other entries' rows are right."""
    with Cache(pkg, "bf16", [100, 230], max_context=600) as c:
        c.fill()
        gen = torch.Generator(device="cuda").manual_seed(2)
        q = torch.randn((84, HQ * D), device="cuda", generator=gen).to(torch.bfloat16)
        for m in (4, 40, 80):
            starts = [0, m, m + 4]
            with pytest.raises(pkg.QkvError) as ei:
                run_attend(c, [None] * 2, q, starts, slots=c.streams, lens=[500, 230])
            assert ei.value.code == 5
            out = torch.full_like(q, -77.0)
            d = [i32(c.streams), i32(starts), i32([500, 230])]
            c.dec.chunk_attend(0, 2, d[0].data_ptr(), d[1].data_ptr(), d[2].data_ptr(), 84, None, q.data_ptr(), out.data_ptr())
            torch.cuda.synchronize()
            with pytest.raises(pkg.QkvError):
                c.dec.sync()
            check_entry(c, c.streams[1], 230, slice(m, m + 4), q, out, visible(226, 4))
            assert (out[m + 4:] == -77).all()


@pytest.mark.parametrize("kv", KINDS)
def test_append_many_rows(pkg, kv):
    """More rows than the SMs take at once, one at a time and together: the same bits; bad and padding rows between."""
    n, lens = 3001, [3001, 3001]
    with Cache(pkg, kv, lens) as c:
        gen = torch.Generator(device="cuda").manual_seed(7)
        qkv = torch.randn((n, QKV), device="cuda", generator=gen)
        axes = torch.randint(-4000, 4000, (3, n), device="cuda", dtype=torch.int32, generator=gen)
        pos = i32(range(n))
        q = torch.full((n, HQ * D), -77.0, device="cuda")
        slots = [c.streams[0]] * n
        slots[1500] = -1
        c.pool.zero_()
        d = i32(slots)
        c.dec.chunk_append(0, n, d.data_ptr(), pos.data_ptr(), axes.data_ptr(), (24, 20, 20), True, qkv.data_ptr(),
                           q.data_ptr(), pkg.F32)
        c.dec.sync()
        one = torch.full((n, HQ * D), -77.0, device="cuda")
        d1 = i32([c.streams[1]] * n)
        picked = [0, 1, 591, 592, 593, 1499, 1501, 2999, 3000]
        for r in picked:
            ax = axes[:, r].contiguous()
            c.dec.chunk_append(0, 1, d1[r:].data_ptr(), pos[r:].data_ptr(), ax.data_ptr(), (24, 20, 20), True,
                               qkv[r].data_ptr(), one[r].data_ptr(), pkg.F32)
        c.dec.sync()
        assert torch.equal(q[picked], one[picked]) and (q[1500] == -77).all() and not (q == -77).all(1)[:1500].any()
        (k0, v0), (k1, v1) = [c.values(0, s, n) for s in c.streams]
        assert torch.equal(k0[picked], k1[picked]) and torch.equal(v0[picked], v1[picked]) and (k0[1500] == 0).all()
        want, mag = append_oracle(qkv.double()[:, :HQ * D].view(n, HQ, D), torch.tensor(c.qn[0], device="cuda").double(), axes,
                                  axis_of_pairs((24, 20, 20), True))
        rows = torch.arange(n, device="cuda") != 1500
        assert not ((q.double().view(n, HQ, D) - want).abs() > 2.0 ** -19 * mag + 1e-30)[rows].any()


@pytest.mark.parametrize("kv,pages", [("bf16", 70000), ("fp8", 135000)])
def test_pools_past_4_gib(pkg, kv, pages):
    """Pages whose bytes lie past 2^32: append, attention, moves, and copies of more pages than a grid has rows."""
    page_bytes = 65536 if kv == "bf16" else 32768
    with Cache(pkg, kv, [], max_streams=2, spare=pages, max_context=8192) as c, Cache(pkg, kv, [3000, 3000]) as small:
        gen = torch.Generator(device="cuda").manual_seed(7)
        qkv = torch.randn((3000, QKV), device="cuda", generator=gen)
        pos, got = i32(range(3000)), []
        for dec in (c.dec, small.dec):
            if dec is c.dec:
                c.streams = [dec.open() for _ in range(2)]
                for s in c.streams:
                    dec.extend(s, 3000)
                assert (dec.pages(c.streams[0]).astype(np.int64) * page_bytes > 1 << 32).any()
            cache = c if dec is c.dec else small
            slots = i32([cache.streams[0]] * 3000)
            axes = torch.stack([pos] * 3).contiguous()
            q = torch.empty((3000, HQ * D), device="cuda", dtype=torch.bfloat16)
            dec.chunk_append(0, 3000, slots.data_ptr(), pos.data_ptr(), axes.data_ptr(), (24, 20, 20), True, qkv.data_ptr(),
                             q.data_ptr(), pkg.BF16)
            dec.sync()
            chunk = q[-70:].contiguous()
            out = run_attend(cache, [(2930, 70)], chunk, [0, 70])
            run_move(cache, [(cache.streams[0], 5, cache.streams[1], 100, list(range(0, 2800, 7)))])
            got.append((q, out, cache.values(0, cache.streams[0], 3000), [t[100:500] for t in cache.values(0, cache.streams[1], 500)]))
        assert torch.equal(got[0][0], got[1][0])
        for x, y in zip(got[0][2] + got[0][3], got[1][2] + got[1][3]):
            assert torch.equal(x, y)
        check_entry(c, c.streams[0], 3000, slice(0, 70), got[0][0][-70:], got[0][1], visible(2930, 70))
        n = pages // 2 - 1000
        perm = np.random.default_rng(1).permutation(pages)
        src, dst = i32(perm[:n]), i32(perm[n:2 * n])
        # a few bytes of each source page tell it from the others
        raw_pool = c.pool.view(torch.uint8).view(pages, page_bytes)
        mark = torch.randint(0, 256, (n, 64), device="cuda", dtype=torch.uint8, generator=gen)
        raw_pool[src.long(), :32] = mark[:, :32]
        raw_pool[src.long(), -32:] = mark[:, 32:]
        c.dec.pages_copy(n, src.data_ptr(), dst.data_ptr())
        c.dec.sync()
        assert torch.equal(raw_pool[dst.long(), :32], mark[:, :32]) and torch.equal(raw_pool[dst.long(), -32:], mark[:, 32:])
        probe = torch.randperm(n, device="cuda", generator=gen)[:500]
        assert torch.equal(raw_pool[dst.long()[probe]], raw_pool[src.long()[probe]])
        if c.scales is not None:
            sc = c.scales.view(torch.int32)[0]
            assert torch.equal(sc[dst.long()], sc[src.long()])


def test_two_handles_at_once(pkg):
    """Calls of two handles on two streams, in flight together, give what they give alone."""
    chunks = [[(900, 9), (40, 130)], [(1500, 30), (10, 2), (333, 70)]]
    with Cache(pkg, "bf16", [b + m for b, m in chunks[0]]) as a, Cache(pkg, "fp8", [b + m for b, m in chunks[1]]) as b:
        caches, work = (a, b), []
        for c, ch in zip(caches, chunks):
            c.fill()
            starts = [sum(m for _, m in ch[:j]) for j in range(len(ch) + 1)]
            gen = torch.Generator(device="cuda").manual_seed(2)
            q = torch.randn((starts[-1], HQ * D), device="cuda", generator=gen).to(torch.bfloat16)
            alone = run_attend(c, ch, q, starts)
            check_attend(c, ch, q, starts, alone)
            lists = [i32(c.streams), i32(starts), i32([base + m for base, m in ch])]
            work.append((c, len(ch), lists, q, alone, [torch.full_like(q, -77.0) for _ in range(20)], torch.cuda.Stream()))
        torch.cuda.synchronize()
        for k in range(20):
            for c, n, lists, q, _, outs, st in work:
                c.dec.chunk_attend(0, n, *[t.data_ptr() for t in lists], q.shape[0], None, q.data_ptr(), outs[k].data_ptr(),
                                   st.cuda_stream)
        torch.cuda.synchronize()
        for c, _, _, _, alone, outs, _ in work:
            c.dec.sync()
            assert all(torch.equal(o, alone) for o in outs)
