"""Cases of the chunk operators of the paged KV cache: their plain forms, the calls a user makes of them, and
their definitions in 64 bits.

Four operators, used together when a stream is continued, branched or verified several tokens at a time:

- append: QK-norm, rotary embedding with a position per axis (time, height, width), K and V into the pages;
- attend: attention of a chunk of new tokens of each stream over its pages, causal or by a draft-tree mask;
- copy:   whole pages copied inside the pool, every layer;
- move:   the accepted tokens of a draft copied to consecutive positions of their stream, every layer.
"""
import math
import random

import torch

own = False

D, HQ, HKV, PAGE = 128, 16, 8, 16
GROUP = HQ // HKV
QKV = (HQ + 2 * HKV) * D
THETA, EPS = 1.0e6, 1.0e-6
LAYERS = 28
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp8": torch.uint8, "e4i8": torch.uint8}


# ---- cases ----

def _attend(streams, chunk_lo, chunk_hi, context_lo, context_hi, kv, tree, shape_seed):
    return dict(op="attend", streams=streams, chunk_lo=chunk_lo, chunk_hi=chunk_hi, context_lo=context_lo,
                context_hi=context_hi, kv=kv, tree=tree, shape_seed=shape_seed)


def _append(rows, kv, interleaved, offset):
    return dict(op="append", rows=rows, kv=kv, interleaved=interleaved, offset=offset)


def _copy(pages, layers, kv):
    return dict(op="copy", pages=pages, layers=layers, kv=kv)


def _move(streams, draft, keep_hi, layers, kv, shape_seed):
    return dict(op="move", streams=streams, draft=draft, keep_hi=keep_hi, layers=layers, kv=kv, shape_seed=shape_seed)


def listed():
    return [
        # one interactive request checks a five-token draft on a short transcript: latency
        dict(_attend(1, 5, 5, 512, 512, "bf16", False, 1), name="verify_one"),
        # a serving batch checks draft trees of ragged sizes: the cache is read once, little arithmetic
        dict(_attend(64, 3, 12, 150, 2100, "bf16", True, 2), name="verify_tree_batch"),
        # a few long recordings in the 8-bit cache: the context has to be split over the card
        dict(_attend(6, 1, 8, 9000, 33000, "e4i8", False, 3), name="verify_long_8bit"),
        # further audio segments of ragged sizes join their streams, e4m3 cache
        dict(_attend(24, 17, 390, 400, 3000, "fp8", False, 4), name="segments_ragged_fp8"),
        # a long prompt taken in pieces: one piece on a long context, bound by arithmetic
        dict(_attend(1, 2048, 2048, 16000, 16000, "bf16", False, 5), name="piece_of_long_prompt"),
        # a draft of a few tokens is appended: latency
        dict(_append(7, "bf16", True, 5000), name="append_draft"),
        # a segment of a few hundred rows, f32 cache and queries
        dict(_append(777, "f32", False, 200), name="append_segment_f32"),
        # the rows of a whole prompt batch, far along the time axis
        dict(_append(16384, "bf16", True, 100000), name="append_prompts"),
        # the last, partly filled pages of a few forked streams
        dict(_copy(5, LAYERS, "bf16"), name="copy_fork_pages"),
        # the pages of a prefix, or a compaction
        dict(_copy(480, LAYERS, "bf16"), name="copy_prefix"),
        # one stream keeps the accepted path of its draft tree
        dict(_move(1, 8, 5, LAYERS, "bf16", 6), name="keep_one"),
        # a serving batch does
        dict(_move(64, 12, 8, LAYERS, "bf16", 7), name="keep_batch"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "append", "copy", "move"])
    if kind == "attend":
        kv = rng.choice(["bf16", "bf16", "fp8", "e4i8"])
        chunk_hi = _log_int(rng, 1, 2048)
        chunk_lo = rng.randint(max(1, chunk_hi // 8), chunk_hi)
        context_hi = _log_int(rng, 1, 32000)
        context_lo = rng.randint(max(0, context_hi // 10), context_hi)
        streams = _log_int(rng, 1, 96)
        most = work(listed()[4])["flops"]
        while True:
            case = _attend(streams, chunk_lo, chunk_hi, context_lo, context_hi, kv,
                           chunk_hi <= 64 and rng.random() < 0.5, rng.randrange(1 << 30))
            if streams == 1 or (work(case)["flops"] <= most and streams * (context_hi + chunk_hi) <= 200000
                                and streams * chunk_hi * (context_hi + chunk_hi) <= 3.4e7):
                break
            streams = max(1, streams // 2)
        if work(case)["flops"] > most:
            case["context_lo"], case["context_hi"] = context_lo // 3, context_hi // 3
        return case
    if kind == "append":
        return _append(_log_int(rng, 1, 16384), rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.5,
                       _log_int(rng, 1, 200000))
    if kind == "copy":
        return _copy(_log_int(rng, 1, 480), rng.choice([1, 2, LAYERS]), "bf16")
    return _move(_log_int(rng, 1, 64), rng.randint(9, 16), rng.randint(1, 9), rng.choice([1, 2, LAYERS]), "bf16",
                 rng.randrange(1 << 30))


def _shape(case):
    """Per stream: tokens before the chunk and tokens of the chunk (attend), or kept tokens (move)."""
    rng = random.Random(case["shape_seed"])
    if case["op"] == "attend":
        return [(rng.randint(case["context_lo"], case["context_hi"]), rng.randint(case["chunk_lo"], case["chunk_hi"]))
                for _ in range(case["streams"])]
    out = []
    for _ in range(case["streams"]):
        base = rng.randint(0, 40)
        keep = sorted(rng.sample(range(case["draft"]), rng.randint(1, min(case["keep_hi"], case["draft"]))))
        out.append((base, keep))
    return out


def _tree_masks(case, chunks):
    """Per chunk row, the bits of the chunk's tokens it sees: itself and its ancestors in a random tree."""
    rng = random.Random(case["shape_seed"] + 1)
    rows = []
    for _, m in chunks:
        own_rows = []
        for j in range(m):
            parent = own_rows[rng.randrange(j)] if j else 0
            own_rows.append(parent | (1 << j))
        rows += own_rows
    return rows


def work(case):
    elem = {"f32": 4, "bf16": 2, "fp8": 1, "e4i8": 1}[case["kv"]]
    token = 2 * HKV * (D * elem + (4 if elem == 1 else 0))
    if case["op"] == "attend":
        chunks = _shape(case)
        rows = sum(m for _, m in chunks)
        if case["tree"]:
            pairs = sum(bin(b).count("1") for b in _tree_masks(case, chunks)) + sum(c * m for c, m in chunks)
        else:
            pairs = sum(c * m + m * (m + 1) // 2 for c, m in chunks)
        return {"bytes": sum(c + m for c, m in chunks) * token + 2 * rows * HQ * D * 2, "flops": 4 * HQ * D * pairs}
    if case["op"] == "append":
        n = case["rows"]
        return {"bytes": n * (QKV * 4 + HQ * D * elem + token), "flops": n * (HQ + HKV) * D * 8}
    if case["op"] == "copy":
        return {"bytes": 2 * case["pages"] * case["layers"] * PAGE * token, "flops": 0}
    kept = sum(len(k) for _, k in _shape(case))
    return {"bytes": 2 * kept * case["layers"] * token, "flops": 0}


# ---- inputs ----

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(shape, seed, dtype=torch.float32):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    gen, step = _gen(seed), 1 << 26   # in pieces: a pool may hold a billion elements
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, device="cuda", generator=gen)
    return out


def _tables(lens, step):
    """Pages of streams that grow in turns, as a pool in use hands them out."""
    tables, have, page = [[] for _ in lens], [0] * len(lens), 0
    turns = []
    while any(h < n for h, n in zip(have, lens)):
        for s, n in enumerate(lens):
            if have[s] < n:
                have[s] = min(n, have[s] + step)
                turns.append((s, have[s]))
                while len(tables[s]) * PAGE < have[s]:
                    tables[s].append(page)
                    page += 1
    return tables, page, turns


def _pool(case, layers, pages, seed):
    """[layers, pages, K|V, head, token, dim] and, for the 8-bit caches, a scale per stored vector."""
    shape = (layers, pages, 2, HKV, PAGE, D)
    if case["kv"] in ("bf16", "f32"):
        return _normal(shape, seed, DTYPES[case["kv"]]), None
    x = _normal(shape, seed)
    amax = x.abs().amax(-1, keepdim=True)
    scale = amax / 448.0
    codes = (x / scale).to(torch.float8_e4m3fn).view(torch.uint8)
    if case["kv"] == "e4i8":
        scale[:, :, 1] = amax[:, :, 1] / 127.0
        codes[:, :, 1] = ((x[:, :, 1] / scale[:, :, 1]).round().clamp(-127, 127) + 128).to(torch.uint8)
    return codes, scale[..., 0].contiguous()


def _axis_of_pair(case):
    """Axis of each of the 64 rotation pairs; sections of 24, 20 and 20 pairs, in blocks or interleaved."""
    sections = (24, 20, 20)
    if case["interleaved"]:
        return [i % 3 if i < 3 * sections[i % 3] else 0 for i in range(D // 2)], sections
    return [0] * sections[0] + [1] * sections[1] + [2] * sections[2], sections


def _inputs(case, seed):
    st = {}
    if case["op"] == "attend":
        chunks = _shape(case)
        lens = [c + m for c, m in chunks]
        rows = sum(m for _, m in chunks)
        st["tables"], pages, st["turns"] = _tables(lens, 512)
        st["pool"], st["scales"] = _pool(case, 1, max(pages, 1), seed)
        st["chunks"], st["lens"], st["rows"] = chunks, lens, rows
        st["starts"] = [sum(m for _, m in chunks[:i]) for i in range(len(chunks) + 1)]
        # normed queries with trained-like gains: some rows attend to a few tokens, some to many
        st["q"] = (_normal((rows, HQ * D), seed + 1) * 1.3).to(torch.bfloat16)
        if case["tree"]:
            bits = [b - (1 << 64) if b >> 63 else b for b in _tree_masks(case, chunks)]
            st["mask"] = torch.tensor(bits, dtype=torch.int64, device="cuda")
    elif case["op"] == "append":
        n = case["rows"]
        per = 410   # rows of one stream: the prompt length of the serving configuration
        lens = [min(per, n - i) for i in range(0, n, per)]
        st["lens"] = lens
        st["tables"], pages, st["turns"] = _tables(lens, 64)
        st["pool"], _ = _pool(case, 1, pages, seed)
        st["slot_of"] = [s for s, m in enumerate(lens) for _ in range(m)]
        st["pos_of"] = [t for m in lens for t in range(m)]
        st["page_of"] = torch.tensor([st["tables"][s][t // PAGE] for s, t in zip(st["slot_of"], st["pos_of"])],
                                     device="cuda")
        # text rows count on along all axes together; frames of 4 x 6 patches share a time and span a grid
        t = torch.arange(n, device="cuda") % per
        frame = (t >= 30) & (t < 30 + 360)
        k = t - 30
        axes = torch.stack([torch.where(frame, 30 + k // 24, t), torch.where(frame, 30 + (k % 24) // 6, t),
                            torch.where(frame, 30 + k % 6, t)])
        st["axes"] = (axes + case["offset"]).to(torch.int32)
        st["qkv"] = _normal((n, QKV), seed + 1)
        st["q_norm"] = 1.0 + 0.1 * _normal((D,), seed + 2)
        st["k_norm"] = 1.0 + 0.1 * _normal((D,), seed + 3)
    elif case["op"] == "copy":
        n = case["pages"]
        st["pool"], _ = _pool(case, case["layers"], 2 * n + 3, seed)
        order = torch.randperm(2 * n + 3, device="cuda", generator=_gen(seed + 1))
        st["src"], st["dst"] = order[:n].to(torch.int32), order[n:2 * n].to(torch.int32)
    else:
        # stream i holds the kept text, stream streams + i the draft
        shape = _shape(case)
        st["lens"] = [b + case["draft"] for b, _ in shape] * 2
        st["tables"], pages, st["turns"] = _tables(st["lens"], 64)
        st["pool"], _ = _pool(case, case["layers"], pages, seed)
        st["shape"] = shape
        n = len(shape)
        at = [(i, b + k, b + j) for i, (b, keep) in enumerate(shape) for k, j in enumerate(keep)]
        st["to"] = torch.tensor([(st["tables"][i][p // PAGE], p % PAGE) for i, p, _ in at], device="cuda").T
        st["from"] = torch.tensor([(st["tables"][n + i][p // PAGE], p % PAGE) for i, _, p in at], device="cuda").T
    return st


class _Memory:
    """Device memory of a decoder as an array that torch can wrap; the decoder lives as long as the array."""

    def __init__(self, owner, ptr, nbytes):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (ptr, False), "version": 3}


def _wrap(owner, ptr, shape, dtype):
    nbytes = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
    return torch.as_tensor(_Memory(owner, ptr, nbytes), device="cuda").view(dtype).view(shape)


def _host_lists(*lists):
    """A call's lists, which change from call to call, in pinned host memory; the call uploads them."""
    return [len(x) for x in lists], torch.tensor([v for x in lists for v in x], dtype=torch.int32).pin_memory()


def _upload(lists):
    """One copy to the device: (what keeps it alive, the address of each list)."""
    sizes, host = lists
    dev = host.to("cuda", non_blocking=True)
    return dev, [dev.data_ptr() + 4 * sum(sizes[:i]) for i in range(len(sizes))]


def _own_state(case, st):
    """The same inputs in a decoder handle: its streams, and its pool filled."""
    import __graft_entry__
    pkg = __graft_entry__.load_package()
    kv = {"f32": pkg.F32, "bf16": pkg.BF16, "fp8": pkg.FP8, "e4i8": pkg.E4I8}[case["kv"]]
    layers, pages = st["pool"].shape[:2]
    lens = st.get("lens", [])
    cfg = dict(n_layers=layers, hidden=1024, n_heads=HQ, n_kv_heads=HKV, head_dim=D, intermediate=256, vocab=256,
               rope_theta=THETA, rms_norm_eps=EPS)
    rt = pkg.runtime_config(device=torch.cuda.current_device(), kv_dtype=kv, max_streams=max(len(lens), 1),
                            max_context=max(lens + [PAGE]), max_pages=pages, max_batch_tokens=64)
    norm = {k: (st[k].cpu().numpy() if k in st else torch.ones(D).numpy())[None].repeat(layers, 0)
            for k in ("q_norm", "k_norm")}
    dec = pkg.Decoder.kv_only(cfg, rt, norm["q_norm"], norm["k_norm"])
    streams = [dec.open() for _ in lens]
    grown = [0] * len(lens)
    for s, upto in st.get("turns", []):
        dec.extend(streams[s], upto - grown[s])
        grown[s] = upto
    info = dec.pool_info()
    pool = _wrap(dec, info["pool"], tuple(st["pool"].shape), st["pool"].dtype)
    pool.copy_(st["pool"])
    st["pool"] = pool
    if st.get("scales") is not None:
        _wrap(dec, info["scales"], tuple(st["scales"].shape), torch.float32).copy_(st["scales"])
    st["dec"], st["pkg"] = dec, pkg
    if case["op"] == "attend":
        st["lists"] = _host_lists(streams, st["starts"], lens)
        st["out"] = torch.empty_like(st["q"])
    elif case["op"] == "append":
        st["lists"] = _host_lists([streams[s] for s in st["slot_of"]], st["pos_of"])
        st["q_out"] = torch.empty((case["rows"], HQ * D), dtype=DTYPES[case["kv"]], device="cuda")
    elif case["op"] == "move":
        n, shape = len(st["shape"]), st["shape"]
        st["to_slots"], st["from_slots"] = _i32(streams[:n]), _i32(streams[n:])
        st["bases"] = _i32([b for b, _ in shape])
        st["starts_dev"] = _i32([sum(len(k) for _, k in shape[:i]) for i in range(n + 1)])
        st["keep"] = _i32([j for _, keep in shape for j in keep])
    torch.cuda.synchronize()
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    return _own_state(case, st) if own else st


# ---- one pass ----

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    case, dec = st["case"], st["dec"]
    stream = torch.cuda.current_stream().cuda_stream or None
    if case["op"] == "attend":
        mask = st["mask"].data_ptr() if case["tree"] else None
        keep, (slots, starts, lens) = _upload(st["lists"])
        dec.chunk_attend(0, len(st["lens"]), slots, starts, lens, st["rows"], mask, st["q"].data_ptr(),
                         st["out"].data_ptr(), stream)
        return st["out"]
    if case["op"] == "append":
        keep, (slots, pos) = _upload(st["lists"])
        dec.chunk_append(0, case["rows"], slots, pos, st["axes"].data_ptr(),
                         _axis_of_pair(case)[1], case["interleaved"], st["qkv"].data_ptr(), st["q_out"].data_ptr(),
                         st["pkg"].F32 if case["kv"] == "f32" else st["pkg"].BF16, stream)
        return {"q": st["q_out"], "pool": st["pool"]}
    if case["op"] == "copy":
        dec.pages_copy(case["pages"], st["src"].data_ptr(), st["dst"].data_ptr(), stream)
        return st["pool"]
    dec.tokens_move(len(st["shape"]), st["from_slots"].data_ptr(), st["bases"].data_ptr(), st["to_slots"].data_ptr(),
                    st["bases"].data_ptr(), st["starts_dev"].data_ptr(), st["keep"].numel(), st["keep"].data_ptr(),
                    stream)
    return st["pool"]


def _stream_kv(st, case, s, dtype):
    """K and V of a stream, [tokens, head, dim], as the values the cache stands for."""
    table = torch.tensor(st["tables"][s], device="cuda")
    pages = st["pool"][0, table]
    if case["kv"] in ("fp8", "e4i8"):
        scale = st["scales"][0, table].to(dtype)[..., None]
        k = pages[:, 0].view(torch.float8_e4m3fn).to(dtype) * scale[:, 0]
        v = pages[:, 1]
        v = (v.to(dtype) - 128.0 if case["kv"] == "e4i8" else v.view(torch.float8_e4m3fn).to(dtype)) * scale[:, 1]
    else:
        k, v = pages[:, 0].to(dtype), pages[:, 1].to(dtype)
    n = st["lens"][s]
    return [x.permute(0, 2, 1, 3).reshape(-1, HKV, D)[:n] for x in (k, v)]


def _visible(st, case, s):
    """[chunk, tokens] truth values of the tokens each row of stream s sees."""
    base, m = st["chunks"][s]
    tok = torch.arange(base + m, device="cuda")
    if case["tree"]:
        bits = st["mask"][st["starts"][s]:st["starts"][s + 1], None]
        return (tok < base) | (((bits >> (tok - base).clamp(0, 63)) & 1) == 1)
    return tok[None] <= base + torch.arange(m, device="cuda")[:, None]


def _run_plain(st):
    case = st["case"]
    if case["op"] == "attend":
        out = torch.empty_like(st["q"])
        for s, (_, m) in enumerate(st["chunks"]):
            k, v = _stream_kv(st, case, s, torch.float32)
            r0, r1 = st["starts"][s], st["starts"][s + 1]
            # a kv head serves GROUP query heads: their rows go through one product
            q = st["q"][r0:r1].float().view(m, HKV, GROUP, D).permute(1, 2, 0, 3).reshape(HKV, GROUP * m, D)
            score = (q @ k.permute(1, 2, 0)) / math.sqrt(D)
            score.masked_fill_(~_visible(st, case, s).repeat(GROUP, 1), -math.inf)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            o = (p @ v.transpose(0, 1)) / p.sum(-1, keepdim=True)
            out[r0:r1] = o.view(HKV, GROUP, m, D).permute(2, 0, 1, 3).reshape(m, HQ * D).to(out.dtype)
        return out
    if case["op"] == "append":
        n = case["rows"]
        axis = torch.tensor(_axis_of_pair(case)[0], device="cuda")
        freq = THETA ** (-2.0 * torch.arange(D // 2, device="cuda", dtype=torch.float64) / D)
        angle = st["axes"].T[:, axis].double() * freq
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

        def norm_rotate(x, w):
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
            a, b = x[..., :D // 2], x[..., D // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        q = norm_rotate(st["qkv"][:, :HQ * D].view(n, HQ, D), st["q_norm"])
        k = norm_rotate(st["qkv"][:, HQ * D:(HQ + HKV) * D].view(n, HKV, D), st["k_norm"])
        v = st["qkv"][:, (HQ + HKV) * D:].view(n, HKV, D)
        pool, tok = st["pool"][0], torch.tensor(st["pos_of"], device="cuda") % PAGE
        pool[st["page_of"], 0, :, tok] = k.to(pool.dtype)
        pool[st["page_of"], 1, :, tok] = v.to(pool.dtype)
        return {"q": q.reshape(n, HQ * D).to(pool.dtype), "pool": st["pool"]}
    if case["op"] == "copy":
        st["pool"][:, st["dst"]] = st["pool"][:, st["src"]]
        return st["pool"]
    (tp, tt), (fp, ft) = st["to"], st["from"]
    st["pool"][:, tp, :, :, tt] = st["pool"][:, fp, :, :, ft]
    return st["pool"]


# ---- the definitions in 64 bits ----

def exact(case, seed):
    if case["op"] in ("copy", "move"):
        return None
    st = _inputs(case, seed)
    if case["op"] == "attend":
        out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
        masks = _tree_masks(case, st["chunks"]) if case["tree"] else None
        for s, (base, m) in enumerate(st["chunks"]):
            t = torch.arange(base + m, device="cuda")
            page = torch.tensor(st["tables"][s], device="cuda")[t // PAGE]
            k, v = st["pool"][0, page, 0, :, t % PAGE], st["pool"][0, page, 1, :, t % PAGE]
            if case["kv"] == "e4i8":
                v = v.double() - 128
            if st["scales"] is not None:
                k, v = [x.view(torch.float8_e4m3fn) if x.dtype == torch.uint8 else x for x in (k, v)]
                k = k.double() * st["scales"][0, page, 0, :, t % PAGE, None].double()
                v = v.double() * st["scales"][0, page, 1, :, t % PAGE, None].double()
            first = st["starts"][s]
            hidden = torch.zeros((m, base + m), dtype=torch.bool)
            for j in range(m):
                hidden[j, base + j + 1:] = True
                if masks:
                    hidden[j, base:] = torch.tensor([not masks[first + j] >> b & 1 for b in range(m)])
            hidden = hidden.cuda()
            for h in range(HQ):
                dims = slice(h * D, (h + 1) * D)
                q = st["q"][first:first + m, dims].double()
                logit = torch.einsum("rd,td->rt", q, k[:, h // GROUP].double()) * D ** -0.5
                logit[hidden] = -math.inf
                out[first:first + m, dims] = torch.einsum("rt,td->rd", torch.softmax(logit, 1), v[:, h // GROUP].double())
        return out
    n = case["rows"]
    axis, _ = _axis_of_pair(case)
    turn = torch.empty((n, D // 2), dtype=torch.complex128, device="cuda")
    for i in range(D // 2):
        turn[:, i] = torch.exp(1j * (st["axes"][axis[i]].double() * THETA ** (-i / (D / 2))))

    def rotated(lo, heads, w):
        x = st["qkv"][:, lo:lo + heads * D].double().view(n, heads, D)
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / D + EPS) * w.double()
        z = torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn[:, None]
        return torch.cat([z.real, z.imag], -1)

    pool = st["pool"].double()
    k = rotated(HQ * D, HKV, st["k_norm"])
    v = st["qkv"][:, (HQ + HKV) * D:].double().view(n, HKV, D)
    page, tok = st["page_of"], torch.tensor(st["pos_of"], device="cuda") % PAGE
    for g in range(HKV):
        pool[0, page, 0, g, tok] = k[:, g]
        pool[0, page, 1, g, tok] = v[:, g]
    return {"q": rotated(0, HQ, st["q_norm"]).reshape(n, HQ * D), "pool": pool}
