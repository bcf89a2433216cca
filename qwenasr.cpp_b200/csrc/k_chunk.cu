// Chunks of new tokens over the paged cache: the append with a rotary position
// per axis, copies of whole pages, and moves of single tokens.  (The attention
// of a chunk is k_chunk_attn.cu.)  The reference appends one prompt or one
// token of one stream (text-decoder.cpp:375-433) and has no counterpart of the
// copies.
#include "kernels.h"

#include "kappend.cuh"

namespace qkv {

namespace {

// ---- append ----
//
// For each head vector x of a row's projection: y = x w / sqrt(mean(x^2) + eps)
// (q and k heads; v is stored as it is), then pair i < 64 of y turns by the
// angle pos[axis(i)] theta^(-2i/128).
//
// Bound by memory: 16 KB in, 8 KB (bf16 q and cache) out per row.  A warp takes
// a quarter of a row (8 heads: q low, q high, k or v), two heads at a time, one
// per half-warp.  A lane holds dims 4l..4l+3 and 64+4l..64+4l+3 of a head, so
// both halves of its four rotation pairs are its own: no shuffles, and the four
// (cos, sin) serve all 8 heads.  Warps stay and go through the rows, the next
// row's eight 16-byte loads per lane (and its slot, page and positions) in
// flight while they compute.  16384 rows, L2 cold: 74 us bf16 (5.5 TB/s), 101 us
// f32 (5.3), 98 us 8-bit (3.8; its head vectors' maxima and divisions besides);
// a block per two rows took 7 us more in bf16.
//
// Angles: positions are any int32, and a float product pos x frequency is off
// by pos 2^-24 radians.  So the frequencies are kept in turns (theta^(-2i/128)
// / 2 pi, f64); the product's fraction of a turn is exact to 2^31 2^-53 turns,
// and only that fraction goes to float and sincospif.
struct ChunkAppendDev {
    AppendParams a;
    const int *axes;          // [3][n]
    const double *turns;      // [64]
    unsigned char axis_of[kHeadDim / 2];
    int q_bf16;
};

constexpr int kAppendWarps = 8;   // two rows a block at a time

template <typename TC>
__device__ __forceinline__ void store4(TC *dst, const float (&v)[4], float inv_scale, bool i8) {
    if constexpr (sizeof(TC) == 4) {
        *reinterpret_cast<float4 *>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    } else if constexpr (sizeof(TC) == 2) {
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w |= (i8 ? f_to_u8ex(v[j] * inv_scale) : static_cast<uint32_t>(f_to_e4m3(v[j] * inv_scale))) << (8 * j);
        *reinterpret_cast<uint32_t *>(dst) = w;
    }
}

template <typename TC>
__global__ void __launch_bounds__(kAppendWarps * 32, 2) chunk_append_kernel(const __grid_constant__ ChunkAppendDev p) {
    pdl_trigger();
    const AppendParams &a = p.a;
    const int warp = blockIdx.x * kAppendWarps + (threadIdx.x >> 5), quarter = warp & 3;
    const int lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15;
    const int step = gridDim.x * (kAppendWarps / 4);

    // What all rows of this lane share: norm weights, frequencies and axes of its rotation pairs.
    float w[8];
    double turns[4];
    int axis[4];
    if (quarter < 3) {
        const float4 *nw = reinterpret_cast<const float4 *>(quarter < 2 ? a.q_norm_w : a.k_norm_w);
        *reinterpret_cast<float4 *>(w) = nw[l];
        *reinterpret_cast<float4 *>(w + 4) = nw[16 + l];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            turns[j] = p.turns[4 * l + j];
            axis[j] = p.axis_of[4 * l + j];
        }
    }
    pdl_wait();   // rows and pages come from earlier kernels; weights and frequencies do not

    // A row's quarter: heads 8 quarter + 2 it + half.
    struct Row {
        float4 lo[4], hi[4];
    };
    const float4 *const src0 = reinterpret_cast<const float4 *>(a.qkv) + (quarter * 8 + half) * (kHeadDim / 4) + l;
    auto load_row = [&](int row, Row &r) {
        const float4 *src = src0 + static_cast<size_t>(row) * (kQkvDim / 4);
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            r.lo[it] = __ldcs(src + it * (2 * kHeadDim / 4));
            r.hi[it] = __ldcs(src + it * (2 * kHeadDim / 4) + kHeadDim / 8);
        }
    };
    struct Where {
        int slot, pos, at[3];
    };
    auto load_where = [&](int row, Where &x) {
        x.slot = a.slots[row];
        x.pos = a.positions[row];
#pragma unroll
        for (int k = 0; k < 3; ++k) x.at[k] = p.axes[static_cast<size_t>(k) * a.n + row];
    };
    auto load_page = [&](const Where &x) -> int {
        if (x.slot < 0 || x.slot >= a.max_streams || x.pos < 0 || x.pos / kPageTokens >= a.maxp) return -2;
        return a.page_table[static_cast<size_t>(x.slot) * a.maxp + x.pos / kPageTokens];
    };

    int row = warp >> 2;
    if (row >= a.n) return;
    Row cur;
    Where here, next{};
    load_row(row, cur);
    load_where(row, here);
    if (row + step < a.n) load_where(row + step, next);
    int page = load_page(here);
    for (; row < a.n; row += step) {
        Row ahead;
        int page_ahead = -2;
        Where after = next;
        if (row + step < a.n) {
            load_row(row + step, ahead);
            page_ahead = load_page(next);
        }
        if (row + 2 * step < a.n) load_where(row + 2 * step, after);

        const bool ok = page >= 0 && page < a.n_pages;
        if (!ok && here.slot != -1 && quarter == 0 && lane == 0)
            report_error(a.err, page == -2 || page == -1 ? kErrPosition : kErrPageIndex, kWhereAppend, row, here.pos);
        if (ok) {   // (slot -1 is a padding row)
            float c[4], s[4];
            if (quarter < 3) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int pos = axis[j] == 0 ? here.at[0] : (axis[j] == 1 ? here.at[1] : here.at[2]);
                    const double t = static_cast<double>(pos) * turns[j];
                    sincospif(2.0f * static_cast<float>(t - rint(t)), &s[j], &c[j]);
                }
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                float x[4] = {cur.lo[it].x, cur.lo[it].y, cur.lo[it].z, cur.lo[it].w};
                float y[4] = {cur.hi[it].x, cur.hi[it].y, cur.hi[it].z, cur.hi[it].w};
                if (quarter < 3) {
                    float ss = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) ss += x[j] * x[j] + y[j] * y[j];
#pragma unroll
                    for (int o = 8; o >= 1; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const float r = 1.0f / sqrtf(ss * (1.0f / kHeadDim) + a.eps);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float u = x[j] * r * w[j], v = y[j] * r * w[4 + j];
                        x[j] = u * c[j] - v * s[j];
                        y[j] = v * c[j] + u * s[j];
                    }
                }
                const int head = quarter * 8 + 2 * it + half;   // 0..15 q, 16..23 k, 24..31 v
                if (quarter < 2) {
                    const size_t off = static_cast<size_t>(row) * kQDim + head * kHeadDim + 4 * l;
                    if (p.q_bf16) {
                        __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(a.q16_out) + off;
                        store4(dst, x, 1.0f, false);
                        store4(dst + kHeadDim / 2, y, 1.0f, false);
                    } else {
                        store4(a.q_out + off, x, 1.0f, false);
                        store4(a.q_out + off + kHeadDim / 2, y, 1.0f, false);
                    }
                    continue;
                }
                const int kv = quarter - 2, g = head & (kHkv - 1), tok = here.pos & (kPageTokens - 1);
                const size_t vec = ((static_cast<size_t>(page) * 2 + kv) * kHkv + g) * kPageTokens + tok;
                float inv_scale = 1.0f;
                const bool i8 = kv == 1 && a.v_int8;
                if constexpr (sizeof(TC) == 1) {
                    float amax = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(x[j]), fabsf(y[j])));
#pragma unroll
                    for (int o = 8; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                    // scale and codes as K1 sets them (append_kv_unit)
                    const float scale = vector_scale(amax, i8 ? kI8Max : kE4m3Max);
                    inv_scale = amax > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
                    if (l == 0) a.scales[vec] = scale;
                }
                TC *dst = static_cast<TC *>(a.pool) + vec * kHeadDim + 4 * l;
                store4(dst, x, inv_scale, i8);
                store4(dst + kHeadDim / 2, y, inv_scale, i8);
            }
        }
        cur = ahead;
        here = next;
        next = after;
        page = page_ahead;
    }
}

// ---- page copies ----
//
// Page src[i] -> dst[i] in every layer, with the 8-bit caches' scales.  Bound
// by memory: twice the bytes.  A block moves 16 KB of one (layer, page): four
// 16-byte loads a thread in flight before its stores.
constexpr int kCopyThreads = 256, kCopyVecs = 4;
constexpr size_t kCopyBlockBytes = kCopyThreads * kCopyVecs * sizeof(uint4);

__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(PagesCopyParams p) {
    pdl_trigger();
    pdl_wait();
    uint4 *const pool = reinterpret_cast<uint4 *>(static_cast<uint8_t *>(p.pool) + blockIdx.z * p.layer_bytes);
    const size_t page_vec = p.page_bytes / sizeof(uint4);
    for (int i = blockIdx.y; i < p.n; i += gridDim.y) {
        const int s = p.src ? p.src[i] : p.src0, d = p.dst ? p.dst[i] : p.dst0;
        if (s < 0 || s >= p.n_pages || d < 0 || d >= p.n_pages) {
            if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.z == 0)
                report_error(p.err, kErrPageIndex, kWherePageCopy, i, s < 0 || s >= p.n_pages ? s : d);
            continue;
        }
        const size_t off = blockIdx.x * (kCopyBlockBytes / sizeof(uint4)) + threadIdx.x;
        const uint4 *from = pool + s * page_vec + off;
        uint4 *to = pool + d * page_vec + off;
        uint4 v[kCopyVecs];
#pragma unroll
        for (int k = 0; k < kCopyVecs; ++k) v[k] = __ldcs(from + k * kCopyThreads);
#pragma unroll
        for (int k = 0; k < kCopyVecs; ++k) __stcs(to + k * kCopyThreads, v[k]);
        if (p.scales && blockIdx.x == 0 && threadIdx.x < kPageScales) {
            float *sc = p.scales + blockIdx.z * p.scales_layer_elems;
            sc[static_cast<size_t>(d) * kPageScales + threadIdx.x] = sc[static_cast<size_t>(s) * kPageScales + threadIdx.x];
        }
    }
}
static_assert(kPageScales <= kCopyThreads, "one thread per scale of a page");
static_assert(kPageHalfElems * 2 % kCopyBlockBytes == 0, "a page of any cache type is whole blocks");

// ---- token moves ----
//
// Group i: its k-th listed token, (src_slots[i], src_bases[i] + keep[starts[i]
// + k]), goes to (dst_slots[i], dst_bases[i] + k), in every layer.  Each thread
// owns one 16-byte piece of the token vectors of one (layer, K|V) and takes the
// tokens in order, eight loads before their stores; within one stream, and in
// pages that the two streams share, the list ascends and targets lie at or below
// their sources, so no store reaches a token that is still to be read.  Bound by latency for one stream (a chain of
// three dependent loads), by memory for many.
constexpr int kMoveBatch = 8;

template <int kElem>
__global__ void __launch_bounds__(kHkv * kHeadDim * kElem / 16) tokens_move_kernel(TokensMoveParams p) {
    constexpr int kVec = kHeadDim * kElem / 16;   // 16-byte pieces of a token vector
    pdl_trigger();
    pdl_wait();
    const int grp = blockIdx.y, layer = blockIdx.x >> 1, kv = blockIdx.x & 1;
    const int from_slot = p.src_slots[grp], to_slot = p.dst_slots[grp];
    if (from_slot == -1 || to_slot == -1) return;   // padding group
    const int k0 = p.starts[grp], k1 = p.starts[grp + 1];
    const int from_base = p.src_bases[grp], to_base = p.dst_bases[grp];
    bool bad = from_slot < 0 || from_slot >= p.max_streams || to_slot < 0 || to_slot >= p.max_streams || k0 < 0 ||
               k1 < k0 || k1 > p.rows || from_base < 0 || to_base < 0 || (from_slot == to_slot && to_base > from_base);
    const int *from_pt = p.page_table + static_cast<size_t>(bad ? 0 : from_slot) * p.maxp;
    const int *to_pt = p.page_table + static_cast<size_t>(bad ? 0 : to_slot) * p.maxp;
    const long long limit = static_cast<long long>(p.maxp) * kPageTokens;
    if (!bad) {
        for (int k = k0 + static_cast<int>(threadIdx.x); k < k1; k += blockDim.x) {
            const int t = p.keep[k];
            const long long a = static_cast<long long>(from_base) + t, b = static_cast<long long>(to_base) + (k - k0);
            if (t < 0 || (k > k0 && t <= p.keep[k - 1]) || a >= limit || b >= limit) {
                bad = true;
                break;
            }
            const int pa = from_pt[a / kPageTokens], pb = to_pt[b / kPageTokens];
            if (pa < 0 || pa >= p.n_pages || pb < 0 || pb >= p.n_pages) bad = true;
            // Streams share pages at equal places only: is the target's page a page of the source stream, too?
            if (to_base > from_base && pb == from_pt[b / kPageTokens]) bad = true;
        }
    }
    if (__syncthreads_or(bad)) {   // every block of the group decides alike: nothing of it moves
        if (threadIdx.x == 0 && blockIdx.x == 0) report_error(p.err, kErrRowBounds, kWhereTokenMove, grp, from_base);
        return;
    }
    uint4 *const pool = reinterpret_cast<uint4 *>(static_cast<uint8_t *>(p.pool) + layer * p.layer_bytes);
    float *const scales = kElem == 1 ? p.scales + layer * p.scales_layer_elems : nullptr;
    const int g = threadIdx.x / kVec, c = threadIdx.x % kVec;
    auto vec = [&](const int *pt, int t) {   // (page, K|V, head, token) of token t of a stream
        return ((static_cast<size_t>(pt[t / kPageTokens]) * 2 + kv) * kHkv + g) * kPageTokens + t % kPageTokens;
    };
    for (int k = k0; k < k1; k += kMoveBatch) {
        uint4 v[kMoveBatch];
        float sc[kMoveBatch];
#pragma unroll
        for (int j = 0; j < kMoveBatch; ++j) {
            if (k + j < k1) {
                const size_t at = vec(from_pt, from_base + p.keep[k + j]);
                v[j] = pool[at * kVec + c];
                if (kElem == 1 && c == 0) sc[j] = scales[at];
            }
        }
#pragma unroll
        for (int j = 0; j < kMoveBatch; ++j) {
            if (k + j < k1) {
                const size_t at = vec(to_pt, to_base + (k + j - k0));
                pool[at * kVec + c] = v[j];
                if (kElem == 1 && c == 0) scales[at] = sc[j];
            }
        }
    }
}

}  // namespace

cudaError_t launch_chunk_append(const ChunkAppendParams &p, int kv_dtype, int num_sms, cudaStream_t st) {
    if (p.a.n <= 0) return cudaSuccess;
    ChunkAppendDev d{};
    d.a = p.a;
    d.axes = p.axes;
    d.turns = p.turns;
    memcpy(d.axis_of, p.axis_of, sizeof d.axis_of);
    d.q_bf16 = p.q_bf16;
    d.a.v_int8 = kv_dtype == kKvE4I8 ? 1 : 0;
    const size_t blocks = (static_cast<size_t>(p.a.n) * 4 + kAppendWarps - 1) / kAppendWarps, full = 2 * static_cast<size_t>(num_sms);
    const dim3 grid(static_cast<unsigned>(blocks < full ? blocks : full));
    const dim3 block(kAppendWarps * 32);
    switch (kv_dtype) {
        case kKvF32: return launch_pdl(chunk_append_kernel<float>, grid, block, 0, st, d);
        case kKvBF16: return launch_pdl(chunk_append_kernel<__nv_bfloat16>, grid, block, 0, st, d);
        case kKvFP8:
        case kKvE4I8: return launch_pdl(chunk_append_kernel<uint8_t>, grid, block, 0, st, d);
        default: return cudaErrorInvalidValue;
    }
}

cudaError_t launch_pages_copy(const PagesCopyParams &p, int n_layers, cudaStream_t st) {
    if (p.n <= 0) return cudaSuccess;
    const dim3 grid(static_cast<unsigned>(p.page_bytes / kCopyBlockBytes), static_cast<unsigned>(p.n < 65535 ? p.n : 65535),
                    static_cast<unsigned>(n_layers));
    return launch_pdl(pages_copy_kernel, grid, dim3(kCopyThreads), 0, st, p);
}

cudaError_t launch_tokens_move(const TokensMoveParams &p, int kv_dtype, int n_layers, cudaStream_t st) {
    if (p.n <= 0) return cudaSuccess;
    const dim3 grid(static_cast<unsigned>(2 * n_layers), static_cast<unsigned>(p.n));
    switch (kv_elem_bytes(kv_dtype)) {
        case 4: return launch_pdl(tokens_move_kernel<4>, grid, dim3(kHkv * kHeadDim * 4 / 16), 0, st, p);
        case 2: return launch_pdl(tokens_move_kernel<2>, grid, dim3(kHkv * kHeadDim * 2 / 16), 0, st, p);
        default: return launch_pdl(tokens_move_kernel<1>, grid, dim3(kHkv * kHeadDim / 16), 0, st, p);
    }
}

}  // namespace qkv
