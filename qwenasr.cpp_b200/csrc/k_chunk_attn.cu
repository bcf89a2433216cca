// Attention of a chunk of new tokens of each stream over its pages: the chunk's
// queries see the tokens before the chunk and, inside it, the tokens up to
// their own (or those of a draft-tree mask).
//
// out[r] = sum_k softmax_k(q_r . k / sqrt(128)) v over the visible tokens; zero
// where none is visible.  bf16 and 8-bit caches, tensor cores (tcgen05, TMEM).
//
// Tiles.  A query tile is 128 MMA rows: 64 queries x the two q heads of a kv
// head g (row 2 i + h), so a K/V tile of 128 keys (8 pages) is fetched once for
// both heads.  S = Q K^T and O += P V are 128 x 128 x 128 each; S and O lie in
// TMEM, P goes back into S's columns as bf16 and is the A operand of P V from
// there.  Two lanes (a softmax warpgroup, an S/P region and an O region each)
// take turns on the tensor cores, so that one lane's MMAs run under the other's
// softmax:
//   pair       (more than 64 queries) the lanes hold query tiles q0 and q0 + 64
//              and both go over every key tile;
//   alternate  (at most 64 queries) both lanes hold the one query tile, lane 0
//              takes the even key tiles of the segment and lane 1 the odd ones;
//              their (max, sum, O) are joined at the segment's end.  A short
//              chunk is bound by reading its context; with half the tiles each,
//              the two lanes' latencies overlap.
//
// Work split.  A unit is (stream, kv head, 128-query block), its work w T: T
// key tiles, w = 2 in pair mode and 1 in alternate mode.  All units laid end to
// end are cut into equal parts, one per CTA (one CTA per SM), wherever the cuts
// fall; a unit cut into pieces leaves (max, sum, unnormalised O) per piece in
// the workspace, and a second kernel joins them in order.  The cuts follow
// from the lengths in device memory alone, so a captured call serves other
// lengths.  Every role walks its CTA's segments by the same arithmetic.
//
// Softmax: thread = row.  P is taken against a reference maximum that moves
// only when a tile exceeds it by more than 2^8 (then O and the sum are
// rescaled); so P <= 2^8, rounded to bf16 once (2^-9 of the weight on average),
// the sum kept in f32 from the unrounded values.  8-bit caches: the codes are
// exact in bf16; a key's scale multiplies its scores, a value's scale its P.
//
// Roles: warps 0..3 loaders (cp.async into the swizzled tiles; 8-bit codes are
// converted on the way), warps 4..7 lane 0, warps 8..11 lane 1, warp 12 MMA.
// All waits bounded.
#include "kernels.h"

#include "ktc.cuh"

namespace qkv {

namespace {

constexpr int kKeys = 128;                 // keys of a tile
constexpr int kQueries = 64;               // queries of a query tile
constexpr int kMmaWarp = 12;
constexpr int kThreads = 13 * 32;
constexpr uint32_t kTmemCols = 512;        // S0 [0,128), S1 [128,256), O0 [256,384), O1 [384,512)
constexpr uint32_t kTmemO = 256;
constexpr float kRescaleLog2 = 8.0f;
constexpr int kMinCost = 2;                // least work of a CTA (tiles of alternate mode)
constexpr int kPieceRows = 256;            // rows of a workspace piece (pair mode: both lanes)

// K and V tiles in flight; 8-bit caches hold raw tiles besides (kRaw) and the
// scales of kScaleRing tiles.
template <bool k8> struct Layout {
    static constexpr int kStages = k8 ? 3 : 5;
    static constexpr int kRaw = k8 ? 3 : 0;
    static constexpr int kLag = 3;         // bf16: tiles issued ahead of the one signalled (< kStages)
    static constexpr int kScaleRing = 4;
    static constexpr size_t kStageOff = 2 * static_cast<size_t>(kTileBytes);
    static constexpr size_t kRawOff = kStageOff + kStages * static_cast<size_t>(kTileBytes);
    static constexpr size_t kScaleOff = kRawOff + kRaw * static_cast<size_t>(kTileBytes / 2);
    static constexpr size_t kRawScaleOff = kScaleOff + (k8 ? kScaleRing * 2 * kKeys * sizeof(float) : 0);
    static constexpr size_t kTailOff = kRawScaleOff + kRaw * 2 * kKeys * sizeof(float);
};

struct Tail {
    uint64_t q_full[2], q_empty[2], full[5], empty[5], s_full[2], p_full[2], pv_done[2], epi_done, x_ready, mma_done;
    uint64_t scale_full[4];                // 8-bit: the scales of a tile are in the ring
    float2 ml[2][128];                     // alternate mode: (max, sum) of each lane's rows
    long long warp_sum[kThreads / 32];
    int warp_max[kThreads / 32];
    long long pre0;                        // work before entry i0, where this CTA's part starts
    int i0, runmax0;
    uint32_t tmem;
    int failed;
};
static_assert(Layout<false>::kTailOff + sizeof(Tail) <= 227 * 1024, "bf16 layout");
static_assert(Layout<true>::kTailOff + sizeof(Tail) <= 227 * 1024, "8-bit layout");

// ---- work split ----

// One listed chunk: its rows, and the work of one kv head.
struct Entry {
    int slot, first, m, base, nb;
    long long head_cost;
    bool bad;
};

__device__ __forceinline__ int block_queries(const Entry &e, int b) { return min(2 * kQueries, e.m - b * 2 * kQueries); }
__device__ __forceinline__ int block_tiles(const Entry &e, int b) {
    return static_cast<int>((static_cast<long long>(e.base) + min(e.m, (b + 1) * 2 * kQueries) + kKeys - 1) / kKeys);
}

// runmax: the largest end of the entries before i; rows that overlap an
// earlier entry's make the later one bad.
__device__ __forceinline__ Entry load_entry(const ChunkAttendParams &p, int i, int runmax) {
    Entry e;
    e.slot = __ldg(p.slots + i);
    e.first = __ldg(p.starts + i);
    const int next = __ldg(p.starts + i + 1), len = __ldg(p.lens + i);
    const bool in = e.first >= 0 && next >= e.first && next <= p.rows && e.first >= runmax;
    e.m = in ? next - e.first : 0;
    e.bad = e.slot != -1 && (!in || e.slot < 0 || e.slot >= p.max_streams || len < e.m ||
                             (static_cast<long long>(len) + kPageTokens - 1) / kPageTokens > p.maxp ||
                             (p.mask && e.m > 64));
    if (e.slot == -1 || e.bad) e.m = 0;
    e.base = len - e.m;
    e.nb = (e.m + 2 * kQueries - 1) / (2 * kQueries);
    e.head_cost = 0;
    if (e.nb > 0) {
        const long long full = e.nb - 1, p0 = (static_cast<long long>(e.base) + kKeys - 1) / kKeys;
        // full blocks end on a multiple of 128 queries: T_b = p0 + b + 1
        e.head_cost = 2 * (full * p0 + full * (full + 1) / 2) +
                      static_cast<long long>(block_queries(e, e.nb - 1) > kQueries ? 2 : 1) * block_tiles(e, e.nb - 1);
    }
    return e;
}

struct Segment {
    int slot, g, row0, nq, q0pos, base, len_end;   // query rows row0.., the first at position q0pos; keys [0, len_end)
    int t0, t1;                                    // key tiles
    bool pair, first, last;                        // holds the unit's first / last tile
    long long ustart;
    int tiles;                                     // of the unit
};

struct Walk {
    Entry e;
    int i, runmax, g, b;
    long long x, x1, ustart;

    __device__ __forceinline__ void start(const ChunkAttendParams &p, const Tail *t, long long from, long long to) {
        x = from;
        x1 = to;
        if (x >= x1) return;
        i = t->i0;
        runmax = t->runmax0;
        e = load_entry(p, i, runmax);
        long long rem = x - t->pre0;
        g = static_cast<int>(rem / e.head_cost);
        rem -= g * e.head_cost;
        b = 0;
        while (b < e.nb - 1) {
            const long long c = 2ll * block_tiles(e, b);
            if (rem < c) break;
            rem -= c;
            ++b;
        }
        ustart = x - rem;
    }
    __device__ __forceinline__ bool next(const ChunkAttendParams &p, Segment &s) {
        while (x < x1) {
            while (g == kHkv || e.m == 0) {        // the next entry with work
                runmax = max(runmax, __ldg(p.starts + i + 1));
                if (++i >= p.n) return false;
                e = load_entry(p, i, runmax);
                g = b = 0;
                ustart = x;
            }
            const int cnt = block_queries(e, b), w = cnt > kQueries ? 2 : 1;
            s.tiles = block_tiles(e, b);
            const long long uend = ustart + static_cast<long long>(w) * s.tiles;
            s.t0 = static_cast<int>((x - ustart + w - 1) / w);
            s.t1 = static_cast<int>(min(static_cast<long long>(s.tiles), (x1 - ustart + w - 1) / w));
            s.slot = e.slot;
            s.g = g;
            s.row0 = e.first + b * 2 * kQueries;
            s.nq = cnt;
            s.base = e.base;
            s.q0pos = e.base + b * 2 * kQueries;
            // with a mask a row may see any token of its chunk; causal blocks end at their last query
            s.len_end = s.q0pos + cnt;
            s.pair = w == 2;
            s.first = s.t0 == 0;
            s.last = s.t1 == s.tiles;
            s.ustart = ustart;
            x = uend;
            ustart = uend;
            if (++b == e.nb) {
                b = 0;
                ++g;
            }
            if (s.t0 < s.t1) return true;
        }
        return false;
    }
};

// Tiles of lane L in a segment: in pair mode lane 0's queries may end a tile
// earlier.
__device__ __forceinline__ int lane_tiles(const Segment &s, int lane) {
    const int n = s.t1 - s.t0;
    if (!s.pair) return (n + 1 - lane) >> 1;
    if (lane == 1) return n;
    return max(0, min(s.t1, (s.q0pos + kQueries + kKeys - 1) / kKeys) - s.t0);
}

// ---- loading ----

__device__ __forceinline__ uint32_t bf16x2_mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t bf16x2_sub(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Four e4m3 codes -> bf16, exactly: sign, exponent and mantissa bits moved to
// their places in a bf16 read 2^-120 of the value (biases 7 and 127), codes
// below the normal range included; 0x7B80 is 2^120.
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t a = __byte_perm(w, 0, 0x1404), b = __byte_perm(w, 0, 0x3424);   // each byte atop 16 bits
    lo = bf16x2_mul(((a & 0x7f007f00u) >> 4) | (a & 0x80008000u), 0x7B807B80u);
    hi = bf16x2_mul(((b & 0x7f007f00u) >> 4) | (b & 0x80008000u), 0x7B807B80u);
}
// Four excess-128 bytes -> bf16, exactly: 0x4300 | (u & 127) is 128 + (u & 127);
// less 256 where u < 128, less 128 (0x4380 with bit 7 cleared) elsewhere.
__device__ __forceinline__ void u8x4_to_bf16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t a = __byte_perm(w, 0, 0x4140), b = __byte_perm(w, 0, 0x4342);
    lo = bf16x2_sub((a & 0x007f007fu) | 0x43004300u, 0x43804380u ^ (a & 0x00800080u));
    hi = bf16x2_sub((b & 0x007f007fu) | 0x43004300u, 0x43804380u ^ (b & 0x00800080u));
}

template <int N> __device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async4(void *dst, const void *src, uint32_t src_bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(src_bytes)
                 : "memory");
}

// Order of the loader's items in a segment of n tiles: K_0, then K_{i+1}, V_i
// for every i (the MMA order), V_{n-1} last; each takes the next stage.
__device__ __forceinline__ uint32_t item_of_k(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ uint32_t item_of_v(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }

template <bool k8>
__global__ void __launch_bounds__(kThreads, 1) chunk_attn_kernel(const __grid_constant__ ChunkAttendParams p) {
    using L = Layout<k8>;
    extern __shared__ uint8_t smem_raw[];
    pdl_trigger();
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint32_t dyn_bytes;
    asm("mov.u32 %0, %%dynamic_smem_size;" : "=r"(dyn_bytes));
    if (static_cast<size_t>(smem - smem_raw) + L::kTailOff + sizeof(Tail) > dyn_bytes) {
        if (threadIdx.x == 0) report_error(p.err, kErrRowBounds, kWhereChunkAttn, -1, static_cast<int>(dyn_bytes));
        pdl_wait();
        return;
    }
    Tail *const tail = reinterpret_cast<Tail *>(smem + L::kTailOff);
    float *const scale_ring = reinterpret_cast<float *>(smem + L::kScaleOff);   // [tile % 4][K|V][key]
    volatile int *const failed = &tail->failed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tail->q_full[b], 128);
            mbar_init(&tail->q_empty[b], 1);
            mbar_init(&tail->s_full[b], 1);
            mbar_init(&tail->p_full[b], 128);
            mbar_init(&tail->pv_done[b], 1);
        }
        for (int b = 0; b < L::kStages; ++b) {
            mbar_init(&tail->full[b], 128);
            mbar_init(&tail->empty[b], 1);
        }
        mbar_init(&tail->epi_done, 256);
        mbar_init(&tail->x_ready, 256);
        mbar_init(&tail->mma_done, 1);
        for (int b = 0; b < L::kScaleRing; ++b) mbar_init(&tail->scale_full[b], 128);
        tail->failed = 0;
        tail->i0 = -1;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail->tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    pdl_wait();   // the entries, q rows and pages come from earlier kernels and copies

    // ---- this CTA's part [x0, x1) of the work: running maximum of the ends, then running sum of the costs ----
    const int per = (p.n + kThreads - 1) / kThreads, e0 = tid * per, e1 = min(p.n, e0 + per);
    int mx = 0;
    for (int i = e0; i < e1; ++i) mx = max(mx, __ldg(p.starts + i + 1));
    int mx_inc = mx;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, mx_inc, o);
        if (lane >= o) mx_inc = max(mx_inc, v);
    }
    if (lane == 31) tail->warp_max[warp] = mx_inc;
    __syncthreads();
    int runmax = __shfl_up_sync(0xffffffffu, mx_inc, 1);
    if (lane == 0) runmax = 0;
    for (int w = 0; w < warp; ++w) runmax = max(runmax, tail->warp_max[w]);
    const int runmax_first = runmax;
    long long sum = 0;
    for (int i = e0; i < e1; ++i) {
        const Entry e = load_entry(p, i, runmax);
        if (e.bad && blockIdx.x == 0) report_error(p.err, kErrRowBounds, kWhereChunkAttn, i, e.first);
        sum += kHkv * e.head_cost;
        runmax = max(runmax, __ldg(p.starts + i + 1));
    }
    long long inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) tail->warp_sum[warp] = inc;
    __syncthreads();
    long long pre = inc - sum, total = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) pre += tail->warp_sum[w];
        total += tail->warp_sum[w];
    }
    const long long parts = max(1ll, min(static_cast<long long>(gridDim.x), total / kMinCost));
    const long long x0 = blockIdx.x < parts ? blockIdx.x * total / parts : 0;
    const long long x1 = blockIdx.x < parts ? (blockIdx.x + 1) * total / parts : 0;
    runmax = runmax_first;
    for (int i = e0; i < e1; ++i) {
        const long long c = kHkv * load_entry(p, i, runmax).head_cost;
        if (pre <= x0 && x0 < pre + c) {
            tail->i0 = i;
            tail->pre0 = pre;
            tail->runmax0 = runmax;
        }
        pre += c;
        runmax = max(runmax, __ldg(p.starts + i + 1));
    }
    if (tid == 0) p.splits[blockIdx.x].c_last = -1;   // no unit starts here and goes on elsewhere (so far)
    __syncthreads();
    fence_after();
    const uint32_t tmem = tail->tmem;

    Walk walk;
    Segment s;
    walk.start(p, tail, x0, x1);

    if (warp < 4) {
        // ================= loaders =================
        const int t = tid;
        uint32_t u = 0, q_fill[2] = {0, 0}, tile_no = 0;
        int qb = 1;
        bool ok = true;
        // bf16: barriers of the items issued and not yet signalled, oldest first.
        // 8-bit: the items in the raw ring instead, as scale slot x 2 + K|V.
        uint64_t *pend[L::kLag] = {};
        uint32_t meta[3] = {0, 0, 0};
        int waiting = 0;
        uint32_t u_conv = 0;
        auto signal_all = [&]() {
            cp_async_wait<0>();
            fence_async_smem();
#pragma unroll
            for (int j = 0; j < L::kLag; ++j) {
                if (pend[j]) mbar_arrive(pend[j]);
                pend[j] = nullptr;
            }
        };
        auto wait_empty = [&](uint64_t *bar, uint32_t par) -> bool {
            if (mbar_try_wait(bar, par)) return true;
            if constexpr (!k8) signal_all();   // what was issued must not wait with us
            if (wait_bar(bar, par, failed)) return true;
            if (!*failed) report_error(p.err, kErrWaitTimeout, kWhereChunkAttn, blockIdx.x, static_cast<int>(u));
            *failed = 1;
            return false;
        };
        auto issued = [&](uint64_t *bar) {     // bf16: bar is signalled once its copies have landed
            cp_async_commit();
            cp_async_wait<L::kLag>();
            if (pend[0]) {
                fence_async_smem();
                mbar_arrive(pend[0]);
            }
#pragma unroll
            for (int j = 0; j + 1 < L::kLag; ++j) pend[j] = pend[j + 1];
            pend[L::kLag - 1] = bar;
        };
        // 8-bit: convert the oldest raw tile into its stage.
        auto convert = [&]() -> bool {
            const uint32_t stage = u_conv % L::kStages, slot = u_conv % (L::kRaw ? L::kRaw : 1);
            if (!wait_empty(&tail->empty[stage], ((u_conv / L::kStages) & 1u) ^ 1u)) return false;
            uint8_t *dst = smem + L::kStageOff + stage * kTileBytes;
            const uint8_t *raw = smem + L::kRawOff + slot * (kTileBytes / 2);
            const uint32_t mt = meta[0];
            const bool i8 = (mt & 1u) && p.v_int8;
            const int c = t & 7;
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                const uint4 w = *reinterpret_cast<const uint4 *>(raw + (m * 128 + t) * 16);
                uint32_t h[8];
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (i8) u8x4_to_bf16(ws[k], h[2 * k], h[2 * k + 1]);
                    else e4m3x4_to_bf16(ws[k], h[2 * k], h[2 * k + 1]);
                }
                const int r = (t >> 3) + 16 * m;
                uint8_t *blk = dst + (c >> 2) * kBlkBytes;
                const uint4 a = make_uint4(h[0], h[1], h[2], h[3]), b = make_uint4(h[4], h[5], h[6], h[7]);
                // lanes of the second block start with their odd chunk: no two of 8 lanes meet in a bank
                const bool odd = c & 4;
                *reinterpret_cast<uint4 *>(blk + swz(r, 2 * (c & 3) + (odd ? 1 : 0))) = odd ? b : a;
                *reinterpret_cast<uint4 *>(blk + swz(r, 2 * (c & 3) + (odd ? 0 : 1))) = odd ? a : b;
            }
            if (!(mt & 1u)) {   // a K tile brings both scales of its tokens
                const float *rs = reinterpret_cast<const float *>(smem + L::kRawScaleOff) + slot * 2 * kKeys;
                scale_ring[(mt >> 1) * 2 * kKeys + t] = rs[t] * p.scale_log2;
                scale_ring[(mt >> 1) * 2 * kKeys + kKeys + t] = rs[kKeys + t];
                mbar_arrive(&tail->scale_full[mt >> 1]);
            }
            fence_async_smem();
            mbar_arrive(&tail->full[stage]);
            ++u_conv;
            meta[0] = meta[1];
            meta[1] = meta[2];
            --waiting;
            return true;
        };
        while (ok && walk.next(p, s) && !*failed) {
            const int *pt = p.page_table + static_cast<size_t>(s.slot) * p.maxp;
            const int key_pages = (s.len_end + kPageTokens - 1) / kPageTokens;
            // Q rows: row 2 i + h, 256 bytes each; rows past the queries are not read by anyone
            for (int j = 0; ok && j < (s.pair ? 2 : 1); ++j) {
                qb = s.pair ? j : qb ^ 1;
                if constexpr (k8) {
                    // Q may be held by tiles that still lie unconverted here
                    if (!mbar_try_wait(&tail->q_empty[qb], (q_fill[qb] & 1u) ^ 1u)) {
                        cp_async_wait<0>();
                        while (ok && waiting > 0) ok = convert();
                    }
                }
                if (!(ok = ok && wait_empty(&tail->q_empty[qb], (q_fill[qb] & 1u) ^ 1u))) break;
                ++q_fill[qb];
                const int rows = 2 * min(kQueries, s.nq - j * kQueries);
                uint8_t *dst = smem + qb * kTileBytes + ((t & 15) >> 3) * kBlkBytes;
                const uint16_t *src = p.q + static_cast<size_t>(s.row0 + j * kQueries) * kQDim + 2 * s.g * kHeadDim + 8 * (t & 15);
#pragma unroll
                for (int m = 0; m < 16; ++m) {
                    const int row = (t >> 4) + 8 * m;
                    if (row < rows)
                        cp_async16(dst + swz(row, t & 7), src + static_cast<size_t>(row >> 1) * kQDim + (row & 1) * kHeadDim, 16u);
                }
                if constexpr (k8) {
                    cp_async_commit();
                    cp_async_wait<0>();
                    fence_async_smem();
                    mbar_arrive(&tail->q_full[qb]);
                } else {
                    issued(&tail->q_full[qb]);
                }
            }
            if (!ok) break;
            const int n = s.t1 - s.t0;
            // pages of the tile whose K / V comes next: V runs one tile behind K
            int pg_k[8], pg_v[8];
            auto pages = [&](int kt, int (&pg)[8]) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int pi = kt * 8 + k;
                    pg[k] = __ldg(pt + (pi < key_pages ? pi : 0));
                }
            };
            auto load = [&](int kt, int kv, const int (&pg)[8], uint32_t scale_slot) -> bool {
                const int live_keys = s.len_end - kt * kKeys;   // of this tile; the rest reads as zero
                bool bad = false;
                if constexpr (!k8) {
                    const uint32_t stage = u % L::kStages;
                    if (!wait_empty(&tail->empty[stage], ((u / L::kStages) & 1u) ^ 1u)) return false;
                    uint8_t *dst = smem + L::kStageOff + stage * kTileBytes + ((t & 15) >> 3) * kBlkBytes + swz(t >> 4, t & 7);
                    const uint8_t *src = static_cast<const uint8_t *>(p.pool) + (kv * kHkv + s.g) * (kPageTokens * kHeadDim * 2) +
                                         (t >> 4) * (kHeadDim * 2) + (t & 15) * 16;
#pragma unroll
                    for (int m = 0; m < 16; ++m) {
                        const int page = pg[m >> 1], r = (t >> 4) + 8 * m;
                        const bool in = page >= 0 && page < p.n_pages, live = r < live_keys;
                        bad = bad || (live && !in);
                        cp_async16(dst + m * 1024,
                                   src + static_cast<size_t>(in ? page : 0) * (kPageHalfElems * 4) + (m & 1) * (8 * kHeadDim * 2),
                                   live && in ? 16u : 0u);
                    }
                    issued(&tail->full[stage]);
                } else {
                    if (waiting == L::kRaw && !convert()) return false;
                    const uint32_t slot = u % (L::kRaw ? L::kRaw : 1);
                    uint8_t *raw = smem + L::kRawOff + slot * (kTileBytes / 2);
                    const uint8_t *src = static_cast<const uint8_t *>(p.pool) + (kv * kHkv + s.g) * (kPageTokens * kHeadDim) +
                                         (t >> 3) * kHeadDim + (t & 7) * 16;
#pragma unroll
                    for (int m = 0; m < 8; ++m) {
                        const int page = pg[m], r = (t >> 3) + 16 * m;
                        const bool in = page >= 0 && page < p.n_pages, live = r < live_keys;
                        bad = bad || (live && !in);
                        cp_async16(raw + (m * 128 + t) * 16, src + static_cast<size_t>(in ? page : 0) * (kPageHalfElems * 2),
                                   live && in ? 16u : 0u);
                    }
                    if (kv == 0) {
                        const int pi = kt * 8 + (t >> 4), page = __ldg(pt + (pi < key_pages ? pi : 0));
                        const bool in = page >= 0 && page < p.n_pages;
                        const float *sc = p.scales + (static_cast<size_t>(in ? page : 0) * 2 * kHkv + s.g) * kPageTokens + (t & 15);
                        float *rs = reinterpret_cast<float *>(smem + L::kRawScaleOff) + slot * 2 * kKeys + t;
                        const uint32_t live = in && t < live_keys ? 4u : 0u;
                        cp_async4(rs, sc, live);
                        cp_async4(rs + kKeys, sc + kHkv * kPageTokens, live);
                    }
                    cp_async_commit();
                    // the raw ring's tiles but the oldest may still be in flight when that one is converted
                    const uint32_t mt = scale_slot * 2 + kv;
                    if (waiting == 0) meta[0] = mt;
                    else if (waiting == 1) meta[1] = mt;
                    else meta[2] = mt;
                    if (++waiting == L::kRaw) cp_async_wait<(L::kRaw > 0 ? L::kRaw - 1 : 0)>();
                }
                ++u;
                if (bad) {
                    report_error(p.err, kErrPageIndex, kWhereChunkAttn, s.row0, kt);
                    *failed = 1;
                    return false;
                }
                return true;
            };
            pages(s.t0, pg_k);
            ok = load(s.t0, 0, pg_k, tile_no % L::kScaleRing);
            for (int i = 0; ok && i < n; ++i) {
#pragma unroll
                for (int k = 0; k < 8; ++k) pg_v[k] = pg_k[k];
                if (i + 1 < n) {
                    pages(s.t0 + i + 1, pg_k);
                    ok = load(s.t0 + i + 1, 0, pg_k, (tile_no + i + 1) % L::kScaleRing);
                }
                ok = ok && load(s.t0 + i, 1, pg_v, (tile_no + i) % L::kScaleRing);
            }
            tile_no += n;
        }
        if constexpr (k8) {
            cp_async_wait<0>();
            while (ok && waiting > 0) ok = convert();
        } else {
            signal_all();
        }
        cp_async_wait<0>();   // no copy outlives the CTA
    } else if (warp == kMmaWarp) {
        // ================= MMA issuer =================
        if (lane == 0) {
            bool ok = true;
            uint32_t u0 = 0, q_use[2] = {0, 0}, p_cnt[2] = {0, 0}, seg = 0;
            int qb = 1;
            while (ok && walk.next(p, s)) {
                const int n = s.t1 - s.t0;
                const int n_l[2] = {lane_tiles(s, 0), lane_tiles(s, 1)};
                int qbuf[2];
                if (s.pair) {
                    qb = 1;
                    qbuf[0] = 0;
                    qbuf[1] = 1;
                } else {
                    qb ^= 1;
                    qbuf[0] = qbuf[1] = qb;
                }
                for (int b = 0; b < 2; ++b) {
                    if (!(s.pair || b == qb)) continue;
                    ok = ok && wait_bar(&tail->q_full[b], q_use[b] & 1u, failed);
                    ++q_use[b];
                }
                if (!ok) break;
                auto stage_of = [&](uint32_t item) { return (u0 + item) % L::kStages; };
                auto wait_item = [&](uint32_t item) {
                    return wait_bar(&tail->full[(u0 + item) % L::kStages], ((u0 + item) / L::kStages) & 1u, failed);
                };
                // S of the lane's tile from K stage `stage`
                auto issue_s = [&](int l, uint32_t stage) {
                    fence_after();
                    const uint32_t aQ = smem_u32(smem + qbuf[l] * kTileBytes);
                    const uint32_t aK = smem_u32(smem + L::kStageOff + stage * kTileBytes);
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk) {
                        const uint32_t off = static_cast<uint32_t>(kk >> 2) * kBlkBytes;
                        const uint64_t step = 2ull * static_cast<uint64_t>(kk & 3);
                        mma(tmem + l * 128u, desc_kmajor(aQ + off) + step, desc_kmajor(aK + off) + step, idesc_s<false>(), kk > 0);
                    }
                    commit(&tail->s_full[l]);
                };
                auto issue_pv = [&](int l, uint32_t stage, bool acc) -> bool {
                    if (!wait_bar(&tail->p_full[l], p_cnt[l] & 1u, failed)) return false;
                    ++p_cnt[l];
                    fence_after();
                    const uint32_t aV = smem_u32(smem + L::kStageOff + stage * kTileBytes);
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk)
                        mma_ta(tmem + kTmemO + l * 128u, tmem + l * 128u + 8u * kk, desc_mnmajor(aV + static_cast<uint32_t>(kk) * 2048u),
                               idesc_pv<false>(), (acc || kk > 0) ? 1 : 0);
                    commit(&tail->pv_done[l]);
                    return true;
                };
                auto q_done = [&]() {   // the segment's last S is issued
                    commit(&tail->q_empty[s.pair ? 0 : qb]);
                    if (s.pair) commit(&tail->q_empty[1]);
                };
                // first tiles
                if (!(ok = wait_item(0))) break;
                if (s.pair) {
                    if (n_l[0] > 0) issue_s(0, stage_of(0));
                    issue_s(1, stage_of(0));
                    commit(&tail->empty[stage_of(0)]);
                } else {
                    issue_s(0, stage_of(0));
                    commit(&tail->empty[stage_of(0)]);
                    if (n > 1) {
                        if (!(ok = wait_item(1))) break;
                        issue_s(1, stage_of(1));
                        commit(&tail->empty[stage_of(1)]);
                    }
                }
                if (n == (s.pair ? 1 : (n > 1 ? 2 : 1))) q_done();
                // the previous segment's O has been read
                if (seg > 0 && !(ok = wait_bar(&tail->epi_done, (seg - 1) & 1u, failed))) break;
                for (int i = 0; ok && i < n; ++i) {
                    const uint32_t vi = item_of_v(i, n);
                    if (!(ok = wait_item(vi))) break;
                    if (s.pair) {
                        const bool more = i + 1 < n;
                        const uint32_t ki = item_of_k(i + 1);
                        if (i < n_l[0]) {
                            if (!(ok = issue_pv(0, stage_of(vi), i > 0))) break;
                            if (i + 1 < n_l[0]) {
                                if (!(ok = wait_item(ki))) break;
                                issue_s(0, stage_of(ki));
                            }
                        }
                        if (!(ok = issue_pv(1, stage_of(vi), i > 0))) break;
                        commit(&tail->empty[stage_of(vi)]);
                        if (more) {
                            if (!(ok = wait_item(ki))) break;
                            issue_s(1, stage_of(ki));
                            commit(&tail->empty[stage_of(ki)]);
                            if (i + 2 == n) q_done();
                        }
                    } else {
                        if (!(ok = issue_pv(i & 1, stage_of(vi), i > 1))) break;
                        commit(&tail->empty[stage_of(vi)]);
                        if (i + 2 < n) {
                            const uint32_t ki = item_of_k(i + 2);
                            if (!(ok = wait_item(ki))) break;
                            issue_s(i & 1, stage_of(ki));
                            commit(&tail->empty[stage_of(ki)]);
                            if (i + 3 == n) q_done();
                        }
                    }
                }
                u0 += 2 * n;
                ++seg;
            }
            if (!ok) {
                if (!*failed) report_error(p.err, kErrWaitTimeout, kWhereChunkAttn, blockIdx.x, 1 << 21);
                *failed = 1;
            }
            // Every MMA issued has completed before TMEM is freed (error path too).
            commit(&tail->mma_done);
            mbar_wait(&tail->mma_done, 0, kWaitLimitCycles);
        }
        __syncwarp();
    } else {
        // ================= softmax and epilogue: lane l, thread = row =================
        const int l = (warp - 4) >> 2, quad = warp & 3, r = 32 * quad + lane, h = r & 1;
        const uint32_t lane_addr = tmem + (static_cast<uint32_t>(32 * quad) << 16);
        const uint32_t tS = lane_addr + l * 128u, tO = lane_addr + kTmemO + l * 128u;
        uint32_t cnt = 0, xcnt = 0, tile_no = 0;
        bool go = true;
        while (walk.next(p, s)) {
            const int n = s.t1 - s.t0, mine = lane_tiles(s, l);
            const int qoff = s.pair ? kQueries * l : 0;
            const int nq = min(kQueries, s.nq - qoff);
            const bool active = 32 * quad < 2 * nq;   // the warp holds a row of a query
            const int i = min(r >> 1, max(nq - 1, 0));
            const int pos_min = s.q0pos + qoff, pos = pos_min + i;
            unsigned long long bits = 0;
            if (p.mask && active) {
                bits = p.mask[s.row0 + qoff + i];
                if (s.nq < 64) bits &= (1ull << s.nq) - 1ull;
            }
            float m_ref = -INFINITY, l_run = 0.0f;
            for (int k = 0; k < mine; ++k) {
                const int ti = s.pair ? k : 2 * k + l, kt = s.t0 + ti;
                go = wait_bar(&tail->s_full[l], cnt & 1u, failed);
                if (!__all_sync(0xffffffffu, go)) break;
                fence_after();
                if (active) {
                    const uint32_t slot = (tile_no + ti) % L::kScaleRing;
                    const float *ks = scale_ring + slot * 2 * kKeys, *vs = ks + kKeys;
                    if constexpr (k8) {
                        go = wait_bar(&tail->scale_full[slot], ((tile_no + ti) / L::kScaleRing) & 1u, failed);
                        if (!__all_sync(0xffffffffu, go)) break;
                    }
                    // keys a row sees, 32 at a time; a tile that every row sees whole needs none of it
                    const bool masked = kt * kKeys + kKeys - 1 > (p.mask ? s.base - 1 : pos_min);
                    auto seen = [&](int c) -> uint32_t {
                        if (!masked) return 0xffffffffu;
                        const int k0 = kt * kKeys + 32 * c;
                        if (!p.mask) {
                            const int d = pos - k0;
                            return d >= 31 ? 0xffffffffu : (d < 0 ? 0u : (2u << d) - 1u);
                        }
                        const int d = k0 - s.base;   // chunk token of the first key
                        if (d <= -32) return 0xffffffffu;
                        if (d < 0) return ((1u << -d) - 1u) | static_cast<uint32_t>(bits << -d);
                        return d < 64 ? static_cast<uint32_t>(bits >> d) : 0u;
                    };
                    // pass 1: the row's largest score
                    float top = -INFINITY;
                    uint32_t sr[2][32];
                    tmem_ld32_issue(tS, sr[0]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        tmem_wait_ld32(sr[c & 1]);
                        if (c < 3) tmem_ld32_issue(tS + 32u * (c + 1), sr[(c + 1) & 1]);
                        const uint32_t w = seen(c);
                        float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            float4 f = make_float4(1.f, 1.f, 1.f, 1.f);
                            if constexpr (k8) f = *reinterpret_cast<const float4 *>(ks + 32 * c + j);
                            const float fs[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                float v = __uint_as_float(sr[c & 1][j + q]);
                                if constexpr (k8) v *= fs[q];
                                if (masked) v = (w >> (j + q)) & 1u ? v : -INFINITY;
                                t4[q] = fmaxf(t4[q], v);
                            }
                        }
                        top = fmaxf(top, fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])));
                    }
                    if constexpr (!k8) top *= p.scale_log2;
                    // the first chunk again, under the decision about the reference
                    tmem_ld32_issue(tS, sr[0]);
                    float alpha = 1.0f;
                    bool rescale = false;
                    if (k == 0) {
                        m_ref = top;
                    } else if (top > m_ref + kRescaleLog2) {
                        alpha = ex2_approx(m_ref - top);   // 0 where nothing was seen so far
                        m_ref = top;
                        l_run *= alpha;
                        rescale = true;
                    }
                    // P V of the lane's previous tile has completed: O is at rest
                    if (k > 0) go = wait_bar(&tail->pv_done[l], (cnt - 1u) & 1u, failed);
                    if (!__all_sync(0xffffffffu, go)) break;
                    if (__any_sync(0xffffffffu, rescale)) {
                        tmem_wait_ld32(sr[0]);
                        fence_after();
#pragma unroll 1
                        for (int c = 0; c < 4; ++c) {
                            float o[32];
                            tmem_ld32(tO + 32u * c, o);
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] *= alpha;
                            tmem_st32(tO + 32u * c, o);
                        }
                        tmem_wait_st();
                        tmem_ld32_issue(tS, sr[0]);
                    }
                    // pass 2: P into S's first 64 columns; chunk c's 16 columns lie in chunks already read
                    const float sub = m_ref == -INFINITY ? 0.0f : m_ref;
                    float acc[2] = {0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        tmem_wait_ld32(sr[c & 1]);
                        if (c < 3) tmem_ld32_issue(tS + 32u * (c + 1), sr[(c + 1) & 1]);
                        const uint32_t w = seen(c);
                        uint32_t pk[16];
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            float4 f = make_float4(1.f, 1.f, 1.f, 1.f), fv = f;
                            if constexpr (k8) {
                                f = *reinterpret_cast<const float4 *>(ks + 32 * c + j);
                                fv = *reinterpret_cast<const float4 *>(vs + 32 * c + j);
                            }
                            const float fs[4] = {f.x, f.y, f.z, f.w}, fvs[4] = {fv.x, fv.y, fv.z, fv.w};
                            float e[4];
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                float v = __uint_as_float(sr[c & 1][j + q]);
                                v = fmaf(v, k8 ? fs[q] : p.scale_log2, -sub);
                                if (masked) v = (w >> (j + q)) & 1u ? v : -INFINITY;
                                e[q] = ex2_approx(v);
                            }
                            acc[0] += e[0] + e[1];
                            acc[1] += e[2] + e[3];
                            if constexpr (k8) {
#pragma unroll
                                for (int q = 0; q < 4; ++q) e[q] *= fvs[q];
                            }
                            pk[j / 2] = pack_bf16x2(e[0], e[1]);
                            pk[j / 2 + 1] = pack_bf16x2(e[2], e[3]);
                        }
                        tmem_st16(tS + 16u * c, pk);
                    }
                    l_run += acc[0] + acc[1];
                    tmem_wait_st();
                } else if (k > 0) {
                    go = wait_bar(&tail->pv_done[l], (cnt - 1u) & 1u, failed);
                    if (!__all_sync(0xffffffffu, go)) break;
                }
                fence_before();
                mbar_arrive(&tail->p_full[l]);
                ++cnt;
            }
            if (!__all_sync(0xffffffffu, go)) break;
            // the lane's last P V
            if (mine > 0) go = wait_bar(&tail->pv_done[l], (cnt - 1u) & 1u, failed);
            if (!__all_sync(0xffffffffu, go)) break;
            // Where this row goes: its dims [d0, d1) of the output row or of the piece's row.
            const bool whole = s.first && s.last;
            float a0 = 1.0f, a1 = 0.0f, m_tot = m_ref, l_tot = l_run;
            if (!s.pair) {
                // lane 1 has nothing to say for a single tile (and must not: lane 0 may still read its last entry)
                if (mine > 0) tail->ml[l][r] = make_float2(m_ref, l_run);
                fence_before();
                mbar_arrive(&tail->x_ready);
                go = wait_bar(&tail->x_ready, xcnt & 1u, failed);
                ++xcnt;
                if (!__all_sync(0xffffffffu, go)) break;
                const float2 v0 = tail->ml[0][r], v1 = n > 1 ? tail->ml[1][r] : make_float2(-INFINITY, 0.0f);
                m_tot = fmaxf(v0.x, v1.x);
                a0 = v0.y > 0.0f ? ex2_approx(v0.x - m_tot) : 0.0f;
                a1 = v1.y > 0.0f ? ex2_approx(v1.x - m_tot) : 0.0f;
                l_tot = a0 * v0.y + a1 * v1.y;
            }
            fence_after();
            const bool real = r < 2 * nq;
            if (active) {
                const float norm = whole ? (l_tot > 0.0f ? 1.0f / l_tot : 0.0f) : 1.0f;
                a0 *= norm;
                a1 *= norm;
                const int c0 = s.pair ? 0 : 2 * l, c1 = s.pair ? 4 : c0 + 2;   // 32-column chunks
                const uint32_t o0 = s.pair ? tO : lane_addr + kTmemO, o1 = lane_addr + kTmemO + 128u;
                const bool own0 = s.pair ? mine > 0 : true, two = !s.pair && n > 1;
                uint16_t *const out = p.out + static_cast<size_t>(s.row0 + qoff + i) * kQDim + (2 * s.g + h) * kHeadDim;
                const size_t piece = 2 * static_cast<size_t>(blockIdx.x) + (s.first ? 1 : 0);
                const int prow = (s.pair ? 128 * l : 0) + r;
                float *const part = p.part_o + piece * (kPieceRows * kHeadDim) + prow * 4;
#pragma unroll 1
                for (int c = c0; c < c1; ++c) {
                    float o[32];
                    if (own0) {
                        tmem_ld32(o0 + 32u * c, o);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = a0 == 0.0f ? 0.0f : o[j] * a0;
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = 0.0f;
                    }
                    if (two) {
                        float o2[32];
                        tmem_ld32(o1 + 32u * c, o2);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] += a1 == 0.0f ? 0.0f : o2[j] * a1;
                    }
                    if (!real) continue;
                    if (whole) {
#pragma unroll
                        for (int j = 0; j < 32; j += 8)
                            *reinterpret_cast<uint4 *>(out + 32 * c + j) =
                                make_uint4(pack_bf16x2(o[j], o[j + 1]), pack_bf16x2(o[j + 2], o[j + 3]),
                                           pack_bf16x2(o[j + 4], o[j + 5]), pack_bf16x2(o[j + 6], o[j + 7]));
                    } else {
                        // a piece keeps four dims of all its rows together: [dims / 4][row][4]
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<float4 *>(part + static_cast<size_t>(8 * c + j / 4) * (kPieceRows * 4)) =
                                make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    }
                }
                if (!whole && real && (s.pair || l == 0))
                    p.part_ml[piece * kPieceRows + prow] = make_float2(m_tot, l_tot);
            }
            fence_before();
            mbar_arrive(&tail->epi_done);
            if (s.first && !s.last && warp == 4 && lane == 0) {
                // the unit goes on in the CTAs up to the one that holds its last tile
                const long long last = s.ustart + static_cast<long long>(s.pair ? 2 : 1) * (s.tiles - 1);
                p.splits[blockIdx.x] = ChunkSplit{s.row0, s.nq, s.g, s.pair ? 1 : 0,
                                                  static_cast<int>(((last + 1) * parts - 1) / total)};
            }
            tile_no += n;
        }
        if (!go) *failed = 1;
    }
    fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// Joins the pieces of the unit that starts in CTA blockIdx.x and goes on
// elsewhere: o = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p, pieces in order.
// Thread = (row, four dims); rows run fastest, as in the pieces.
constexpr int kJoinThreads = 256;

__global__ void __launch_bounds__(kJoinThreads) chunk_join_kernel(const __grid_constant__ ChunkAttendParams p) {
    pdl_trigger();
    pdl_wait();
    const ChunkSplit d = p.splits[blockIdx.x];
    const int c0 = blockIdx.x;
    if (d.c_last <= c0) return;
    const int rows = 2 * d.nq;   // pair: lane 0's 128 rows, then lane 1's
    for (int w = blockIdx.y * kJoinThreads + threadIdx.x; w < rows * (kHeadDim / 4); w += gridDim.y * kJoinThreads) {
        const int r = w % rows, c = w / rows;
        float m = -INFINITY;
        for (int k = c0; k <= d.c_last; ++k) m = fmaxf(m, p.part_ml[(2 * k + (k == c0 ? 1 : 0)) * kPieceRows + r].x);
        float l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = c0; k <= d.c_last; ++k) {
            const size_t piece = 2 * k + (k == c0 ? 1 : 0);
            const float2 ml = p.part_ml[piece * kPieceRows + r];
            if (!(ml.y > 0.0f)) continue;
            const float a = exp2f(ml.x - m);
            const float4 v = *reinterpret_cast<const float4 *>(p.part_o + piece * (kPieceRows * kHeadDim) +
                                                               static_cast<size_t>(c) * (kPieceRows * 4) + r * 4);
            l += a * ml.y;
            o[0] += a * v.x;
            o[1] += a * v.y;
            o[2] += a * v.z;
            o[3] += a * v.w;
        }
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        uint16_t *out = p.out + static_cast<size_t>(d.row0 + (r >> 1)) * kQDim + (2 * d.g + (r & 1)) * kHeadDim + 4 * c;
        *reinterpret_cast<uint2 *>(out) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
    }
}

template <bool k8> size_t smem_want() { return Layout<k8>::kTailOff + sizeof(Tail) + 1023; }

size_t smem_capped(size_t want, int optin) { return want < static_cast<size_t>(optin) ? want : static_cast<size_t>(optin); }

cudaError_t smem_optin(int *optin) {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    return e != cudaSuccess ? e : cudaDeviceGetAttribute(optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
}

}  // namespace

ChunkWorkspace chunk_workspace(int num_sms) {
    const size_t pieces = 2 * static_cast<size_t>(num_sms);
    return ChunkWorkspace{pieces * kPieceRows * kHeadDim, pieces * kPieceRows, static_cast<size_t>(num_sms)};
}

cudaError_t prepare_chunk_attn() {
    int optin = 0;
    cudaError_t e = smem_optin(&optin);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(chunk_attn_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem_capped(smem_want<false>(), optin)));
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(chunk_attn_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(smem_capped(smem_want<true>(), optin)));
}

cudaError_t launch_chunk_attn(const ChunkAttendParams &p, int kv_dtype, int num_sms, cudaStream_t st) {
    if (p.n <= 0 || p.rows <= 0) return cudaSuccess;
    int optin = 0;
    cudaError_t e = smem_optin(&optin);
    if (e != cudaSuccess) return e;
    if (kv_dtype == kKvBF16)
        e = launch_pdl(chunk_attn_kernel<false>, dim3(num_sms), dim3(kThreads), smem_capped(smem_want<false>(), optin), st, p);
    else if (kv_is_8bit(kv_dtype))
        e = launch_pdl(chunk_attn_kernel<true>, dim3(num_sms), dim3(kThreads), smem_capped(smem_want<true>(), optin), st, p);
    else
        return cudaErrorInvalidValue;
    if (e != cudaSuccess) return e;
    return launch_pdl(chunk_join_kernel, dim3(num_sms, 8), dim3(kJoinThreads), 0, st, p);
}

}  // namespace qkv
