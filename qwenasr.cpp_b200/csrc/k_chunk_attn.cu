// Attention of a chunk of new tokens of each stream over its pages: the chunk's
// queries see the tokens before the chunk and, inside it, the tokens up to
// their own (or those of a draft-tree mask).
//
// out[r] = sum_k softmax_k(q_r . k / sqrt(128)) v over the visible tokens; zero
// where none is visible.  bf16 and 8-bit caches, tensor cores (tcgen05, TMEM).
// A sum of exponentials is 0 only where nothing is visible (or every score is
// -infinity), so every division and skip asks for 0 and lets a NaN, from scores
// of NaN or +infinity, through to its row.
//
// A K/V tile is 128 keys (8 pages) of one kv head g, fetched once for the two q
// heads it serves.  Two lanes (a softmax warpgroup, an S region and an O region
// of TMEM each) take turns on the tensor cores, so that one lane's MMAs run
// under the other's softmax.  A unit, (stream, g, up to 128 queries), runs in
// one of three modes by its number of queries:
//   pair       65..128: each lane holds a query tile of 128 MMA rows (64 queries
//              x 2 heads, row 2 i + h) and both go over every key tile;
//   alternate  17..64: both lanes hold the one query tile, lane 0 takes the even
//              key tiles of the segment and lane 1 the odd ones;
//   thin       1..16: the lanes alternate too, but with keys and queries
//              exchanged, S' = K Q' and O' = V' P' (128 keys x 16 or 32 columns).
// In pair and alternate mode S = Q K', thread = query row; P goes back over S as
// bf16 and is the A operand of P V in TMEM.  That costs a thread 128
// exponentials a tile however few rows are real, which a short chunk, bound by
// reading its context, cannot hide (64 draft trees of 3 to 12 rows on contexts
// of 150 to 2100 tokens: 186 us when thin mode was added, 76 us in it now, 53 us
// to read them); in thin mode a thread has one key and computes 16 or 32.
//
// Work split.  A unit's work is w T: T key tiles, w = 2 in pair mode and 1
// elsewhere.  All units laid end to end are cut into equal parts, one per CTA
// (one CTA per SM), wherever the cuts fall; a unit cut into pieces leaves (max,
// sum, unnormalised O) per piece in the workspace, and a second kernel joins
// them in order.  The cuts follow from the lengths in device memory alone, so a
// captured call serves other lengths.  One warp walks a CTA's segments and
// hands them to the others through a ring in shared memory.
//
// Softmax.  P is taken against a reference that moves only when a tile's scores
// exceed it by more than 2^kRescaleLog2 (thin mode) or its sum leaves the range
// of kSumMax (then O and the sum are rescaled); P, the sum and O are floating-point numbers and lose nothing to a common factor.  P is
// rounded to bf16 once (2^-8 of the weight at most); sums stay in f32 and take
// the unrounded values.  8-bit caches: the codes are exact in bf16; a key's
// scale multiplies its scores, a value's scale its P.
//
// Roles: warps 0..3 lane 0, 4..7 lane 1, one MMA warp, two load warps (TMA: a
// page's 16 keys of a head are a box; one warp K and Q, one V), one that plans
// the segments, and for 8-bit caches eight that convert the raw tiles.  Staging
// the tiles by cp.async from four warps took 2700 cycles per 32 KB and bounded
// every shape; the MMA warp runs its loop as a whole and elects a thread only to
// issue, so that descriptors stay in uniform registers.  What a segment's start
// and end cost was mostly code fetched afresh, so those parts are kept short or
// rolled up.
//
// What bounds it (device time of calls in a graph, L2 warm; cycles by clock64 in
// the MMA warp, fitted as a tile's and a segment's over all segments).
// 2048 bf16 rows on 16000 tokens: 400 000 cycles a CTA, 251 us in bursts of some
// ms (1.14 PFLOP/s), 295 us after seconds at the power cap (0.97).  A pair step
// takes 3200 cycles, of which the tensor cores work 2100 and each softmax warp
// 2060, which is its 128 exponentials a row at the pipe's rate; the rest is one
// lane waiting where neither covers the other.
// Alternate mode, 16 chunks of 40 bf16 rows on 2000 tokens: 41 us, 2200 cycles a
// tile and 7800 a segment.
// The draft trees above: 4.6 TB/s; 1850 cycles a tile and 7500 to 8000 a segment,
// its start and end.
// Six 8-bit contexts of 9000 to 33000 tokens: 98 us, 3.2 TB/s; 2400 cycles a
// tile, of which the converting warps work 864 for each of K and V (with the
// conversion left out, 88 us of what was 101 then).
// 24 ragged segments of 17 to 390 rows on 400 to 3000 tokens: 105 us bf16, 155 us
// e4m3; a pair step of the latter takes 5900 to 6100 cycles, as each softmax
// warp reads two scales a key besides and shares its scheduler with the
// converting warps.
// Five rows on 512 tokens: 9.6 us, a chain of latencies (plan 3300 cycles, K tile
// in place at 7100, P V done at 9200, epilogue 2100, then the join).
// All waits bounded; a softmax warp whose wait ran out goes on without waiting,
// so that the named barriers stay matched.
#include <cuda.h>

#include <type_traits>

#include "kernels.h"

#include "ktc.cuh"

namespace qkv {

namespace {

constexpr int kKeys = 128;                 // keys of a tile
constexpr int kQueries = 64;               // queries of a query tile
constexpr uint32_t kTmemCols = 512;        // S0 [0,128), S1 [128,256), O0 [256,384), O1 [384,512)
constexpr uint32_t kTmemO = 256;
constexpr float kRescaleLog2 = 30.0f;
// Pair and alternate mode: bounds of a sum of 32 or 128 terms, 2^60 and 2^40.  Past kSumMove the reference moves before
// the next tile; only past kSumMax it has to at once.  (O then stays finite for values below 2^67.)
constexpr float kSumMax = 1152921504606846976.0f, kSumMove = 1099511627776.0f;
constexpr int kThinQueries = 16;           // most queries of thin mode
enum Mode { kThin = 0, kAlternate = 1, kPair = 2 };
// The two 32 KB areas before the stages: a query tile each, or area 1 split
// between thin mode's two query buffers (32 rows) and the lanes' P tiles.
constexpr uint32_t kThinQ = kTileBytes, kThinQBytes = 8192, kThinQBlk = 4096;
constexpr uint32_t kThinP = kTileBytes + 16384, kThinPBytes = 8192;
constexpr int kMinCost = 2;                // least work of a CTA (tiles of alternate mode)
static_assert(kMinCost >= 2, "every CTA between a unit's first and last holds one of its tiles");
// Work of a unit besides its tiles, for all modes and cache types: 5000 to 8000 cycles and 1850 to 3200 a tile outside
// pair mode, 9000 to 11500 and 3200 to 6000 a tile (counted double) in it.  Of (2, 3), (3, 6), (5, 9) and (8, 14): 64
// draft trees 80, 80, 76, 76 us; ragged bf16 segments 118, 115, 105, 106; ragged e4m3 160, 162, 155, 163; six long 8-bit
// contexts 97, 97, 98, 99; 16 chunks of 40 rows on 2000 tokens 41, 41, 41, 40; a 2048-row piece 251, 251, 251, 253.
constexpr int kUnitCost = 5, kPairUnitCost = 9;
constexpr int kPieceRows = 256;            // rows of a workspace piece (pair mode: both lanes)

// K and V tiles in flight; 8-bit caches hold raw tiles besides (kRaw) and the
// scales of kScaleRing tiles.
template <bool k8> struct Layout {
    static constexpr int kStages = k8 ? 3 : 5;
    static constexpr int kRaw = k8 ? 3 : 0;
    static constexpr int kScaleRing = 4;
    static constexpr int kConvWarp = 8, kConvWarps = k8 ? 8 : 0;
    static constexpr int kMmaWarp = kConvWarp + kConvWarps;
    static constexpr int kLoadWarp = kMmaWarp + 1;   // K tiles and Q; the next one V tiles
    static constexpr int kPlanWarp = kMmaWarp + 3;
    static constexpr int kWarps = kMmaWarp + 4, kThreads = 32 * kWarps;
    // Registers: the launch gives every thread kRegs (65536 over the threads, in eights); the warpgroups then trade
    // them.  bf16: 12 warps x 168 = 2 x 4 x 208 + 4 x 80 (and some left); 8-bit: 20 x 96 = 2 x 4 x 144 + 3 x 4 x 64.
    static constexpr int kSoftmaxRegs = k8 ? 144 : 208, kOtherRegs = k8 ? 64 : 80, kRegs = k8 ? 96 : 168;
    static_assert(8 * kSoftmaxRegs + (kWarps - 8) * kOtherRegs <= kWarps * kRegs, "register split");
    static constexpr size_t kStageOff = 2 * static_cast<size_t>(kTileBytes);
    static constexpr size_t kRawOff = kStageOff + kStages * static_cast<size_t>(kTileBytes);
    static constexpr size_t kScaleOff = kRawOff + kRaw * static_cast<size_t>(kTileBytes / 2);
    static constexpr size_t kRawScaleOff = kScaleOff + (k8 ? kScaleRing * 2 * kKeys * sizeof(float) : 0);
    static constexpr size_t kTailOff = kRawScaleOff + kRaw * 2 * kKeys * sizeof(float);
};

// ---- work split ----

// One listed chunk: its rows, and the work of one kv head.
struct Entry {
    int slot, first, m, base, nb;
    int head_cost;            // (all work of a call together stays below 2^31: chunk_work_fits)
    bool bad;
};

__device__ __forceinline__ int block_queries(const Entry &e, int b) { return min(2 * kQueries, e.m - b * 2 * kQueries); }
__device__ __forceinline__ int block_tiles(const Entry &e, int b) {
    return static_cast<int>((static_cast<unsigned>(e.base) + min(e.m, (b + 1) * 2 * kQueries) + kKeys - 1) / kKeys);
}

struct RawEntry {
    int slot, first, next, len;
};
__device__ __forceinline__ RawEntry load_raw(const ChunkAttendParams &p, int i) {
    return {__ldg(p.slots + i), __ldg(p.starts + i), __ldg(p.starts + i + 1), __ldg(p.lens + i)};
}

// runmax: the largest end of the entries before it; rows that overlap an
// earlier entry's make the later one bad.
__device__ __forceinline__ Entry make_entry(const ChunkAttendParams &p, const RawEntry &r, int runmax) {
    Entry e;
    e.slot = r.slot;
    e.first = r.first;
    const int next = r.next, len = r.len;
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
        const int full = e.nb - 1, p0 = static_cast<int>((static_cast<unsigned>(e.base) + kKeys - 1) / kKeys);
        // full blocks end on a multiple of 128 queries: T_b = p0 + b + 1
        e.head_cost = 2 * (full * p0 + full * (full + 1) / 2) +
                      (block_queries(e, e.nb - 1) > kQueries ? 2 : 1) * block_tiles(e, e.nb - 1) +
                      kPairUnitCost * full + (block_queries(e, e.nb - 1) > kQueries ? kPairUnitCost : kUnitCost);
    }
    return e;
}

struct alignas(16) Segment {
    int slot, g, row0, nq;            // query rows row0 ..
    int q0pos, base, len_end, mode;   // position of the first query, of the chunk's first token; keys [0, len_end)
    int t0, t1, cols, first;          // key tiles; thin mode's columns (2 nq rounded up to 16); holds the first tile
    int last, c_first, c_last, pad;   // holds the unit's last tile; the CTAs that hold its first and its last
    __device__ __forceinline__ bool pair() const { return mode == kPair; }
};

// Areas that a segment's Q (thin: and P) takes, as a bit set, after a segment
// with `prev`; an alternate segment avoids its predecessor's.
__device__ __forceinline__ uint32_t q_areas(int mode, uint32_t prev) {
    return mode == kPair ? 3u : (mode == kThin ? 2u : (prev & 1u ? 2u : 1u));
}

// Where a CTA's part starts: the entry, the largest end before it, the work before it.
struct Start {
    int i, runmax, pre;
};

// The work cut into equal parts, the first r of them one larger.
struct Cuts {
    int parts, q, r;
    __device__ __forceinline__ int at(int c) const { return c * q + min(c, r); }   // where part c starts
    __device__ __forceinline__ int holder(int pos) const {
        const int lim = r * (q + 1);
        return pos < lim ? static_cast<int>(static_cast<unsigned>(pos) / static_cast<unsigned>(q + 1))
                         : r + static_cast<int>(static_cast<unsigned>(pos - lim) / static_cast<unsigned>(q));
    }
};
__device__ __forceinline__ Cuts cut_work(int total) {
    const int parts = max(1, min(static_cast<int>(gridDim.x), total / kMinCost)), q = total / parts;
    return {parts, q, total - q * parts};
}

constexpr int kSegRing = 4;
struct alignas(16) Tail {
    Segment seg[kSegRing];
    // (reference, sum) of each lane's rows or columns at a segment's end.  Thin mode uses 0..31 and, for its column
    // sums by warp, 64..127; of lane 0, 32..63 for the columns' factors.  Before the first segment: the scan's scratch.
    float2 ml[2][128];
    float thin_ref[2][32];                 // thin mode: the lane's reference per column
    uint64_t q_full[2], q_free[2];         // of a segment, by its parity; q_free: its areas
    uint64_t full[5], empty[5], s_full[2], p_full[2], o_full[2], epi_done, mma_done;
    uint64_t seg_full[kSegRing], seg_empty[kSegRing];
    uint64_t scale_full[4], raw_full[3], raw_empty[3];   // 8-bit
    Start from;
    uint32_t tmem;
    int failed;
    uint32_t issued[5], q_issued;          // last item of each ring slot and last Q, plus one
};
static_assert(Layout<false>::kTailOff + sizeof(Tail) <= 227 * 1024, "bf16 layout");
static_assert(Layout<true>::kTailOff + sizeof(Tail) <= 227 * 1024, "8-bit layout");

// Goes through the segments of a CTA's part [x, x1) of the work.
struct Walk {
    Entry e;
    int i, runmax, g, b;
    int x, x1, ustart;
    Cuts cuts;

    __device__ __forceinline__ void start(const Entry &first, const Start &f, const Cuts &c) {
        cuts = c;
        x = x1 = 0;
        if (static_cast<int>(blockIdx.x) < c.parts) {
            x = c.at(blockIdx.x);
            x1 = c.at(blockIdx.x + 1);
        }
        if (x >= x1) return;
        i = f.i;
        runmax = f.runmax;
        e = first;
        int rem = x - f.pre;
        g = rem / e.head_cost;
        rem -= g * e.head_cost;
        b = 0;
        while (b < e.nb - 1) {
            const int c = 2 * block_tiles(e, b) + kPairUnitCost;
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
                e = make_entry(p, load_raw(p, i), runmax);
                g = b = 0;
                ustart = x;
            }
            const int cnt = block_queries(e, b), w = cnt > kQueries ? 2 : 1;
            const int tiles = block_tiles(e, b);
            // tile t is the CTA's that holds position `at` + w t
            const int at = ustart + (w == 2 ? kPairUnitCost : kUnitCost), uend = at + w * tiles;
            s.t0 = max(0, x - at + w - 1) >> (w - 1);
            s.t1 = min(tiles, max(0, x1 - at + w - 1) >> (w - 1));
            s.slot = e.slot;
            s.g = g;
            s.row0 = e.first + b * 2 * kQueries;
            s.nq = cnt;
            s.base = e.base;
            s.q0pos = e.base + b * 2 * kQueries;
            // with a mask a row may see any token of its chunk; causal blocks end at their last query
            s.len_end = s.q0pos + cnt;
            s.mode = w == 2 ? kPair : (cnt > kThinQueries ? kAlternate : kThin);
            s.cols = cnt > 8 ? 32 : 16;
            s.first = s.t0 == 0;
            s.last = s.t1 == tiles;
            s.c_first = cuts.holder(at);
            s.c_last = cuts.holder(at + w * (tiles - 1));
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
    if (!s.pair()) return (n + 1 - lane) >> 1;
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
// below the normal range included; 0x7B80 is 2^120.  A code times 16 has
// exponent and mantissa in place and the sign at bit 11; 15 times that bit more
// puts it at bit 15.  (Multiplications, because the pipe for shifts and logic is
// the one that a tile's softmax fills.)
__device__ __forceinline__ uint32_t e4m3x2_to_bf16(uint32_t two) {   // one code in the low byte of each half
    const uint32_t y = two * 16u;
    return bf16x2_mul((y & 0x08000800u) * 15u + y, 0x7B807B80u);
}
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    lo = e4m3x2_to_bf16(__byte_perm(w, 0, 0x4140));
    hi = e4m3x2_to_bf16(__byte_perm(w, 0, 0x4342));
}
// Four excess-128 bytes -> bf16, exactly: 0x4300 | (u & 127) is 128 + (u & 127);
// less 256 where u < 128, less 128 (0x4380 with bit 7 cleared) elsewhere.
__device__ __forceinline__ void u8x4_to_bf16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t a = __byte_perm(w, 0, 0x4140), b = __byte_perm(w, 0, 0x4342);
    lo = bf16x2_sub((a & 0x007f007fu) | 0x43004300u, 0x43804380u ^ (a & 0x00800080u));
    hi = bf16x2_sub((b & 0x007f007fu) | 0x43004300u, 0x43804380u ^ (b & 0x00800080u));
}

// One box of a tensor map -> shared memory, completing on `bar`; what lies
// outside the map reads as zero.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// A load that stays where it is written, a tile ahead of its use.
__device__ __forceinline__ int load_early(const int *p) {
    int v;
    asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
template <int kRegs> __device__ __forceinline__ void set_regs_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs> __device__ __forceinline__ void set_regs_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// A value that all lanes hold alike (and >= 0), by way of a warp reduction, whose result the compiler knows to be
// uniform: what MMA and TMA instructions take from uniform registers then needs no transfer each time.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ int uniform(int v) { return static_cast<int>(uniform(static_cast<uint32_t>(v))); }

// Packed pairs of f32 (two lanes of one instruction).
__device__ __forceinline__ uint64_t f2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void un_f2(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Named barriers of a softmax warpgroup (128 threads) and of both (256).
__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("barrier.cta.sync.aligned %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ bool bar_any(int id, int threads, bool pred) {
    int r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred.aligned q, %2, %3, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(static_cast<int>(pred)), "r"(id), "r"(threads)
        : "memory");
    return r != 0;
}
constexpr int kBarLane = 1, kBarBoth = 3;   // ids kBarLane + lane, kBarBoth

// kCols TMEM columns of this thread's lane; usable after tmem_wait_ld_regs.
template <int kCols> __device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[kCols]) {
    static_assert(kCols == 8 || kCols == 16 || kCols == 32, "");
    if constexpr (kCols == 32) {
        tmem_ld32_issue(taddr, r);
    } else if constexpr (kCols == 16) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
            "%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
              "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr));
    } else {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                     : "r"(taddr));
    }
}
template <int kCols> __device__ __forceinline__ void tmem_wait_ld_regs(uint32_t (&r)[kCols]) {
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < kCols; ++j) asm volatile("" : "+r"(r[j]));   // no use moves ahead of the wait
}

// Thin mode's P (bf16, [128 keys][kCols], columns contiguous: MN-major B):
// rows of 32 or 64 bytes, swizzled over 256 or 512 bytes.
__device__ __forceinline__ uint64_t desc_thin_p(uint32_t addr, int cols) {
    return ((addr >> 4) & 0x3FFFull) | (1ull << 16) | (static_cast<uint64_t>(cols) << 32) | (1ull << 46) |
           ((cols == 16 ? 6ull : 4ull) << 61);   // 8-key groups 16 cols bytes apart
}
__device__ __forceinline__ uint32_t idesc_thin(int cols) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(cols >> 3) << 17) | ((128u >> 4) << 24);
}
constexpr uint32_t kIdescTransposeAB = (1u << 15) | (1u << 16);

// Sum of each of kCols registers over the warp's 32 lanes: afterwards v[0]
// holds column lane / (32 / kCols).
template <int kCols> __device__ __forceinline__ void warp_column_sums(float (&v)[kCols], int lane) {
    int o = 16;
#pragma unroll
    for (int cnt = kCols / 2; cnt >= 1; cnt >>= 1, o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int j = 0; j < cnt; ++j) {
            const float send = up ? v[j] : v[j + cnt], keep = up ? v[j + cnt] : v[j];
            v[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    }
    for (; o >= 1; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
}

// Largest of x over the warp (redux on the order-preserving integer image).
__device__ __forceinline__ float warp_max(float x) {
    int i = __float_as_int(x);
    i ^= (i >> 31) & 0x7fffffff;
    i = __reduce_max_sync(0xffffffffu, i);
    i ^= (i >> 31) & 0x7fffffff;
    return __int_as_float(i);
}

// Order of the loader's items in a segment of n tiles: K_0, then K_{i+1}, V_i
// for every i (the MMA order), V_{n-1} last; each takes the next stage.
__device__ __forceinline__ uint32_t item_of_k(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ uint32_t item_of_v(int i, int n) { return i == n - 1 ? 2 * n - 1 : 2 * i + 2; }

// Tensor maps: the layer's pool as [page][K|V x head x token][dim] with boxes of
// 16 tokens x 128 bytes, swizzled, and q as
// [row][head][dim] with boxes of 64 and 16 rows x 2 heads x 64 dims.
struct Maps {
    CUtensorMap kv, q, q_thin;
    CUtensorMap scales;   // 8-bit: [page][K|V][head][token], boxes of one head's K and V scales
};

template <bool k8>
__global__ void __launch_bounds__(Layout<k8>::kThreads, 1)
    chunk_attn_kernel(const __grid_constant__ ChunkAttendParams p, const __grid_constant__ Maps maps) {
    using L = Layout<k8>;
    constexpr int kThreads = L::kThreads, kMmaWarp = L::kMmaWarp;
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
            mbar_init(&tail->q_full[b], 1);
            mbar_init(&tail->q_free[b], 1);
            mbar_init(&tail->s_full[b], 1);
            mbar_init(&tail->p_full[b], 4);      // warps
            mbar_init(&tail->o_full[b], 1);
        }
        for (int b = 0; b < L::kStages; ++b) {
            mbar_init(&tail->full[b], k8 ? 32 * L::kConvWarps : 1);
            mbar_init(&tail->empty[b], 1);
        }
        for (int b = 0; b < kSegRing; ++b) {
            mbar_init(&tail->seg_full[b], 1);
            mbar_init(&tail->seg_empty[b], L::kWarps - 1);   // the other warps
        }
        mbar_init(&tail->epi_done, 8);      // warps
        mbar_init(&tail->mma_done, 1);
        for (int b = 0; b < L::kScaleRing; ++b) mbar_init(&tail->scale_full[b], 128);
        for (int b = 0; b < L::kRaw; ++b) {
            mbar_init(&tail->raw_full[b], 1);
            mbar_init(&tail->raw_empty[b], 32 * L::kConvWarps);
        }
        tail->failed = 0;
        for (int b = 0; b < 5; ++b) tail->issued[b] = 0;
        tail->q_issued = 0;
        tail->from = Start{0, 0, 0};
        fence_mbar_init();
    }
    if (warp == L::kLoadWarp && lane == 0) {
        prefetch_map(&maps.kv);
        prefetch_map(&maps.q);
        prefetch_map(&maps.q_thin);
        if (k8) prefetch_map(&maps.scales);
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tail->tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tail->tmem;
    pdl_wait();   // the entries, q rows and pages come from earlier kernels and copies

    // ---- this CTA's part of the work ----
    // Running maximum of the ends and running sum of the costs over the entries: up to 32 by the plan warp itself (its
    // part of a small call is a chain of latencies, and begins here), more by all threads, kPer to a thread (n <= 1024).
    int total = 0;
    if (p.n > 32) {
        constexpr int kPer = (kAttnMaxRows + kThreads - 1) / kThreads;
        const int e0 = tid * kPer;
        RawEntry raw[kPer];
        int mx = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) raw[k] = e0 + k < p.n ? load_raw(p, e0 + k) : RawEntry{-1, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < kPer; ++k) mx = max(mx, raw[k].next);
        int mx_inc = mx;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, mx_inc, o);
            if (lane >= o) mx_inc = max(mx_inc, v);
        }
        int *const warp_sum = reinterpret_cast<int *>(tail->ml[0]);
        int *const warp_max = reinterpret_cast<int *>(tail->ml[1]);
        if (lane == 31) warp_max[warp] = mx_inc;
        __syncthreads();
        int runmax = __shfl_up_sync(0xffffffffu, mx_inc, 1);
        if (lane == 0) runmax = 0;
        for (int w = 0; w < warp; ++w) runmax = max(runmax, warp_max[w]);
        int cost[kPer], sum = 0;
        int maxes[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            maxes[k] = runmax;
            const Entry e = make_entry(p, raw[k], runmax);
            if (e.bad && blockIdx.x == 0) report_error(p.err, kErrRowBounds, kWhereChunkAttn, e0 + k, e.first);
            cost[k] = kHkv * e.head_cost;
            sum += cost[k];
            runmax = max(runmax, raw[k].next);
        }
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) warp_sum[warp] = inc;
        __syncthreads();
        int pre = inc - sum;
        for (int w = 0; w < L::kWarps; ++w) {
            if (w < warp) pre += warp_sum[w];
            total += warp_sum[w];
        }
        const Cuts cuts = cut_work(total);
        const int x0 = cuts.at(blockIdx.x);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (pre <= x0 && x0 < pre + cost[k]) tail->from = Start{e0 + k, maxes[k], pre};
            pre += cost[k];
        }
        __syncthreads();
    }
    if (tid == 0) p.splits[2 * blockIdx.x].n = p.splits[2 * blockIdx.x + 1].n = 0;   // no unit cut here (so far)

    Segment s;
    uint32_t seg_no = 0;
    // The next segment (the same for every warp); false behind the last one.
    auto next_segment = [&]() -> bool {
        const uint32_t b = seg_no % kSegRing;
        const bool there = __all_sync(0xffffffffu, wait_bar(&tail->seg_full[b], (seg_no / kSegRing) & 1u, failed));
        if (!there) {
            if (lane == 0 && !*failed) report_error(p.err, kErrWaitTimeout, kWhereChunkAttn, blockIdx.x, 1 << 18);
            *failed = 1;
            return false;
        }
        s = tail->seg[b];
        __syncwarp();
        if (lane == 0) mbar_arrive(&tail->seg_empty[b]);
        ++seg_no;
        return s.slot >= 0;
    };

    if (warp >= L::kMmaWarp) {
    set_regs_down<L::kOtherRegs>();
    if (warp == L::kPlanWarp) {
        // ================= plan: the segments, one after the other =================
        Entry mine;
        Start from;
        Cuts cuts;
        if (p.n <= 32) {
            RawEntry raw{-1, 0, 0, 0};
            if (lane < p.n) raw = load_raw(p, lane);
            int mx = raw.next;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, mx, o);
                if (lane >= o) mx = max(mx, v);
            }
            mx = __shfl_up_sync(0xffffffffu, mx, 1);
            const int runmax = lane == 0 ? 0 : max(mx, 0);
            mine = make_entry(p, raw, runmax);
            if (mine.bad && blockIdx.x == 0) report_error(p.err, kErrRowBounds, kWhereChunkAttn, lane, mine.first);
            const int c = kHkv * mine.head_cost;
            int inc = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            cuts = cut_work(__shfl_sync(0xffffffffu, inc, 31));
            const int x0 = cuts.at(blockIdx.x);
            const unsigned has = __ballot_sync(0xffffffffu, inc - c <= x0 && x0 < inc);
            const int i0 = has ? __ffs(has) - 1 : 0;
            from = Start{i0, __shfl_sync(0xffffffffu, runmax, i0), __shfl_sync(0xffffffffu, inc - c, i0)};
            mine.slot = __shfl_sync(0xffffffffu, mine.slot, i0);
            mine.first = __shfl_sync(0xffffffffu, mine.first, i0);
            mine.m = __shfl_sync(0xffffffffu, mine.m, i0);
            mine.base = __shfl_sync(0xffffffffu, mine.base, i0);
            mine.nb = __shfl_sync(0xffffffffu, mine.nb, i0);
            mine.head_cost = __shfl_sync(0xffffffffu, mine.head_cost, i0);
        } else {
            cuts = cut_work(total);
            from = tail->from;
            mine = make_entry(p, load_raw(p, from.i), from.runmax);
        }
        if (lane == 0) {
            Walk walk;
            walk.start(mine, from, cuts);
            bool more = true;
            for (uint32_t k = 0; more; ++k) {
                const uint32_t b = k % kSegRing;
                Segment next;
                more = walk.next(p, next);
                if (!more) next.slot = -1;
                if (!wait_bar(&tail->seg_empty[b], ((k / kSegRing) & 1u) ^ 1u, failed)) {
                    if (!*failed) report_error(p.err, kErrWaitTimeout, kWhereChunkAttn, blockIdx.x, 1 << 17);
                    *failed = 1;
                    break;
                }
                tail->seg[b] = next;
                mbar_arrive(&tail->seg_full[b]);
            }
        }
        __syncwarp();
    } else if (warp >= L::kLoadWarp) {
        // ================= loads =================
        const int kv = warp - L::kLoadWarp;
        constexpr int kRing = k8 ? L::kRaw : L::kStages;
        uint64_t *const ring_full = k8 ? tail->raw_full : tail->full, *const ring_empty = k8 ? tail->raw_empty : tail->empty;
        uint32_t u0 = 0, seg = 0, areas = 0;
        bool ok = true, was_thin = false;
        auto wait = [&](uint64_t *bar, uint32_t par) -> bool {
            const bool done = wait_bar(bar, par, failed);
            if (__all_sync(0xffffffffu, done)) return true;
            if (lane == 0 && !*failed) report_error(p.err, kErrWaitTimeout, kWhereChunkAttn, blockIdx.x, static_cast<int>(u0));
            *failed = 1;
            return false;
        };
        const bool leader = elect_one();
        const uint32_t smem_u = uniform(smem_u32(smem));
        const int ps = lane & 7;   // this lane's page of a tile
        while (ok && next_segment() && !*failed) {
            const int *const pt = p.page_table + static_cast<size_t>(s.slot) * p.maxp;
            const int key_pages = (s.len_end + kPageTokens - 1) / kPageTokens, n = uniform(s.t1 - s.t0);
            auto page_id = [&](int kt) { return kt * 8 + ps < key_pages ? load_early(pt + kt * 8 + ps) : p.n_pages; };
            // Outside the map's pages a box reads as zero: behind the last page, and for a bad id.
            auto checked = [&](int id, int kt) {
                if (static_cast<unsigned>(id) < static_cast<unsigned>(p.n_pages)) return id;
                if (kt * 8 + ps < key_pages) report_error(p.err, kErrPageIndex, kWhereChunkAttn, s.row0, kt);
                return p.n_pages;
            };
            int id_next = page_id(s.t0);
            const int g2 = uniform(2 * s.g), row0 = uniform(s.row0);
            // One thread issues a tile's boxes from warp-uniform page ids: as many lanes issuing one each took 90 cycles
            // a box.
            auto load = [&](int kt, uint32_t u, int id) -> bool {
                const uint32_t slot = u % kRing;
                int ids[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) ids[k] = uniform(ps == k ? id : 0);
                const int y = kv * (kHkv * kPageTokens) + g2 * (kPageTokens / 2);
                if (!wait(&ring_empty[slot], ((u / kRing) & 1u) ^ 1u)) return false;
                uint64_t *const bar = &ring_full[slot];
                if constexpr (!k8) {
                    const uint32_t dst = smem_u + static_cast<uint32_t>(L::kStageOff) + slot * kTileBytes;
                    // V rows behind the last token must be zero (their weight is zero, but not a NaN's product with
                    // it): the page the stream ends in comes by plain loads.
                    const int live = s.len_end - kt * kKeys, rows = live & (kPageTokens - 1), part = live >> 4;
                    const bool mixed = kv == 1 && live < kKeys && rows != 0;
                    if (mixed) {
                        const int page = __shfl_sync(0xffffffffu, id, part);
                        uint8_t *const to = smem + L::kStageOff + slot * kTileBytes;
                        const uint8_t *const from = static_cast<const uint8_t *>(p.pool) +
                                                    ((static_cast<size_t>(page < p.n_pages ? page : 0) * 2 + 1) * kHkv + s.g) *
                                                        (kPageTokens * kHeadDim * 2);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int row = (lane >> 4) + 2 * j, c = lane & 15;
                            const uint4 v = row < rows && page < p.n_pages
                                                ? *reinterpret_cast<const uint4 *>(from + row * (kHeadDim * 2) + c * 16)
                                                : make_uint4(0, 0, 0, 0);
                            *reinterpret_cast<uint4 *>(to + (c >> 3) * kBlkBytes + swz(part * kPageTokens + row, c & 7)) = v;
                        }
                        fence_async_smem();
                        __syncwarp();
                    }
                    if (leader) {
                        mbar_arrive_expect_tx(bar, kTileBytes - (mixed ? kTileBytes / 8 : 0));
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            if (mixed && k == part) continue;
                            tma_load_3d(dst + k * 2048, &maps.kv, 0, y, ids[k], bar);
                            tma_load_3d(dst + kBlkBytes + k * 2048, &maps.kv, 64, y, ids[k], bar);
                        }
                    }
                } else {
                    const uint32_t dst = smem_u + static_cast<uint32_t>(L::kRawOff) + slot * (kTileBytes / 2);
                    const uint32_t dst_s = smem_u + static_cast<uint32_t>(L::kRawScaleOff) + slot * (2 * kKeys * 4);
                    if (leader) {
                        // a K tile brings both scales of its tokens
                        mbar_arrive_expect_tx(bar, kTileBytes / 2 + (kv == 0 ? 2 * kKeys * 4 : 0));
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            tma_load_3d(dst + k * 2048, &maps.kv, 0, y, ids[k], bar);
                            if (kv == 0) tma_load_4d(dst_s + k * (2 * kPageTokens * 4), &maps.scales, 0, g2 >> 1, 0, ids[k], bar);
                        }
                    }
                }
                if (leader) tail->issued[slot] = u + 1;
                __syncwarp();
                return true;
            };
            auto load_q = [&]() -> bool {
                // Q takes the areas of an earlier segment: the one before last has always ended (its Q barrier is
                // reused), the last one if they meet.
                const uint32_t prev = areas;
                areas = q_areas(s.mode, prev);
                const bool meets = (areas & prev) && !(s.mode == kThin && was_thin);
                was_thin = s.mode == kThin;
                if (seg >= 2) ok = wait(&tail->q_free[seg & 1u], ((seg - 2) >> 1) & 1u);
                if (ok && meets && seg >= 1) ok = wait(&tail->q_free[(seg - 1) & 1u], ((seg - 1) >> 1) & 1u);
                // Q rows: row 2 i + h.  Rows behind the unit's queries are some other row's or zero: rows (in thin mode
                // columns) of S that no one reads.
                if (!ok) return false;
                if (leader) {
                    uint64_t *bar = &tail->q_full[seg & 1u];
                    if (s.mode == kThin) {
                        const uint32_t dst = smem_u32(smem) + kThinQ + (seg & 1u) * kThinQBytes;
                        mbar_arrive_expect_tx(bar, 2 * kThinQBlk);
                        tma_load_3d(dst, &maps.q_thin, 0, g2, row0, bar);
                        tma_load_3d(dst + kThinQBlk, &maps.q_thin, 64, g2, row0, bar);
                    } else {
                        const int tiles = s.pair() ? 2 : 1;
                        mbar_arrive_expect_tx(bar, tiles * kTileBytes);
                        for (int j = 0; j < tiles; ++j) {
                            const uint32_t dst = smem_u32(smem) + (s.pair() ? j * kTileBytes : (areas >> 1) * kTileBytes);
                            tma_load_3d(dst, &maps.q, 0, g2, row0 + j * kQueries, bar);
                            tma_load_3d(dst + kBlkBytes, &maps.q, 64, g2, row0 + j * kQueries, bar);
                        }
                    }
                }
                if (leader) tail->q_issued = seg + 1;
                return ok;
            };
            for (int i = 0; ok && i < n; ++i) {
                const int id = checked(id_next, s.t0 + i);
                if (i + 1 < n) id_next = page_id(s.t0 + i + 1);
                ok = load(s.t0 + i, u0 + (kv ? item_of_v(i, n) : item_of_k(i)), id);
                if (i == 0 && kv == 0) ok = ok && load_q();   // its area may have to be waited for; the tile need not
            }
            u0 += 2 * n;
            ++seg;
        }
    } else {
        // ================= MMA issuer =================
        bool ok = true;
        const bool leader = elect_one();
        // Tiles are consumed in the order they are loaded: a running stage and its phase.
        uint32_t st = 0, ph = 0, p_cnt0 = 0, p_cnt1 = 0, seg = 0, areas = 0;
        const uint32_t tmem_u = uniform(tmem), smem_u = uniform(smem_u32(smem));
        auto wait = [&](uint64_t *bar, uint32_t par) { return __all_sync(0xffffffffu, wait_bar(bar, par, failed)) != 0; };
        while (ok && next_segment()) {
            // warp-uniform copies: what the descriptors are made of
            const int n = uniform(s.t1 - s.t0), n0 = uniform(lane_tiles(s, 0)), mode = uniform(s.mode), cols = uniform(s.cols);
            const bool pair = mode == kPair, thin = mode == kThin;
            areas = uniform(q_areas(mode, areas));
            if (!(ok = wait(&tail->q_full[seg & 1u], (seg >> 1) & 1u))) break;
            // the next tile, once it is there
            auto next_tile = [&](uint32_t &stage) -> bool {
                stage = st;
                const bool there = wait(&tail->full[st], ph);
                if (++st == L::kStages) {
                    st = 0;
                    ph ^= 1u;
                }
                return there;
            };
            auto q_done = [&]() {
                if (leader) commit(&tail->q_free[seg & 1u]);
            };
            const uint32_t aQ0 = smem_u + (thin ? kThinQ + (seg & 1u) * kThinQBytes : (pair ? 0u : (areas >> 1) * kTileBytes));
            const uint32_t id_thin = idesc_thin(cols);
            auto free_stage = [&](uint32_t stage) {
                if (leader) commit(&tail->empty[stage]);
            };
            // S of the lane's tile from K stage `stage`
            auto issue_s = [&](int l, uint32_t stage) {
                fence_after();
                const Desc k(desc_kmajor(smem_u + static_cast<uint32_t>(L::kStageOff) + stage * kTileBytes));
                const Desc q(desc_kmajor(aQ0 + (pair ? l * kTileBytes : 0u)));
                if (leader) {
                    if (thin) {
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)
                            mma(tmem_u + l * 128u, k, (kk >> 2) * (kBlkBytes >> 4) + 2 * (kk & 3), q,
                                (kk >> 2) * (kThinQBlk >> 4) + 2 * (kk & 3), id_thin, kk > 0);
                    } else {
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk) {
                            const uint32_t off = (kk >> 2) * (kBlkBytes >> 4) + 2 * (kk & 3);
                            mma(tmem_u + l * 128u, q, off, k, off, idesc_s<false>(), kk > 0);
                        }
                    }
                    commit(&tail->s_full[l]);
                }
                __syncwarp();
            };
            auto issue_pv = [&](int l, uint32_t stage, bool acc, bool last) -> bool {
                const uint32_t par = l ? p_cnt1++ : p_cnt0++;
                if (!wait(&tail->p_full[l], par & 1u)) return false;
                fence_after();
                const Desc v(desc_mnmajor(smem_u + static_cast<uint32_t>(L::kStageOff) + stage * kTileBytes));   // 2 KB per 16 keys
                const uint32_t tO = tmem_u + kTmemO + l * 128u;
                if (leader) {
                    if (thin) {
                        const Desc pt(desc_thin_p(smem_u + kThinP + l * kThinPBytes, cols));
                        const uint32_t p16 = 2u * cols;   // 16 keys of P, in 16-byte units
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)
                            mma(tO, v, kk * 128u, pt, kk * p16, id_thin | kIdescTransposeAB, (acc || kk > 0) ? 1 : 0);
                    } else {
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)
                            mma_ta(tO, tmem_u + l * 128u + 8u * kk, v, kk * 128u, idesc_pv<false>(), (acc || kk > 0) ? 1 : 0);
                    }
                    if (last) commit(&tail->o_full[l]);   // the lane's O of this segment is complete
                }
                __syncwarp();
                return true;
            };
            uint32_t kt = 0, vt = 0;
            // first tiles
            if (!(ok = next_tile(kt))) break;
            if (n0 > 0) issue_s(0, kt);
            if (pair) issue_s(1, kt);
            free_stage(kt);
            if (!pair && n > 1) {
                if (!(ok = next_tile(kt))) break;
                issue_s(1, kt);
                free_stage(kt);
            }
            if (!thin && n <= (pair ? 1 : 2)) q_done();   // Q is read by S alone; thin mode's area holds P, too
            // the previous segment's O has been read
            if (seg > 0 && !(ok = wait(&tail->epi_done, (seg - 1) & 1u))) break;
            if (pair) {
                for (int i = 0; i < n; ++i) {
                    const bool more = i + 1 < n;
                    if (more && !(ok = next_tile(kt))) break;
                    if (!(ok = next_tile(vt))) break;
                    if (i < n0) {
                        if (!(ok = issue_pv(0, vt, i > 0, i + 1 == n0))) break;
                        if (i + 1 < n0) issue_s(0, kt);
                    }
                    if (!(ok = issue_pv(1, vt, i > 0, i + 1 == n))) break;
                    free_stage(vt);
                    if (more) {
                        issue_s(1, kt);
                        free_stage(kt);
                        if (i + 2 == n) q_done();
                    }
                }
            } else {
                for (int i = 0; i < n; ++i) {
                    const int l = i & 1;
                    if (!(ok = next_tile(vt))) break;
                    if (!(ok = issue_pv(l, vt, i > 1, i + 2 >= n))) break;
                    free_stage(vt);
                    if (i + 2 < n) {
                        if (!(ok = next_tile(kt))) break;
                        issue_s(l, kt);
                        free_stage(kt);
                        if (!thin && i + 3 == n) q_done();
                    }
                }
            }
            if (!ok) break;
            if (thin) q_done();
            ++seg;
        }
        if (!ok) {
            if (lane == 0 && !*failed) report_error(p.err, kErrWaitTimeout, kWhereChunkAttn, blockIdx.x, 1 << 21);
            *failed = 1;
        }
        // Every MMA issued has completed before TMEM is freed (error path too).
        if (leader) {
            commit(&tail->mma_done);
            mbar_wait(&tail->mma_done, 0, kWaitLimitCycles);
        }
        __syncwarp();
    }
    } else if (k8 && warp >= L::kConvWarp) {
        set_regs_down<L::kOtherRegs>();
        // ================= 8-bit codes -> bf16 tiles =================
        // Thread: a 16-byte piece of rows row + 32 m.  Eight lanes take four pieces of rows r and r ^ 5, which differ in
        // bits 0 and 2: swizzled, neither their 16-byte reads (pieces c ^ r) nor their writes (2 c ^ r, 2 c + 1 ^ r)
        // meet in a bank.
        constexpr int kRows = 4;
        constexpr uint32_t kRing = k8 ? L::kRaw : 1;
        const int t = tid - 32 * L::kConvWarp, c = (lane & 3) | ((lane >> 1) & 4), pair_no = (t >> 5) * 2 + (lane >> 4);
        const int row0 = (pair_no >> 2) * 8 + (pair_no & 3), row = lane & 4 ? row0 ^ 5 : row0;
        const uint32_t src0 = smem_u32(smem) + static_cast<uint32_t>(L::kRawOff) + swz(row, c);
        const uint32_t dst0 = smem_u32(smem) + static_cast<uint32_t>(L::kStageOff) + (c >> 2) * kBlkBytes + swz(row, 2 * (c & 3));
        const uint32_t dst1 = dst0 ^ 16u;
        uint32_t u = 0, tile_no = 0;
        bool ok = true;
        auto give_up = [&](int where) {
            if (!*failed) report_error(p.err, kErrWaitTimeout, kWhereChunkAttn, blockIdx.x, where);
            *failed = 1;
            return false;
        };
        auto item = [&](int kt, int kv, uint32_t tile) -> bool {
            const uint32_t slot = u % kRing, stage = u % L::kStages;
            if (!wait_bar(&tail->raw_full[slot], (u / kRing) & 1u, failed)) return give_up(1 << 20);
            if (kv == 0 && t < kKeys) {   // a K tile brings both scales of its tokens; none behind the last one
                const float *const rs = reinterpret_cast<const float *>(smem + L::kRawScaleOff) + slot * 2 * kKeys +
                                        (t >> 4) * (2 * kPageTokens) + (t & 15);
                const bool live = kt * kKeys + t < s.len_end;
                const uint32_t ring = tile % L::kScaleRing;
                // A hidden key's score, -infinity, is multiplied by this, so it must not be zero: a vector stored with
                // scale 0 gets the least f32 instead, which moves a finite score by 2^-21 at most.
                const float fk = rs[0] * p.scale_log2;
                scale_ring[ring * 2 * kKeys + t] = !live ? 1.0f : (fk != 0.0f ? fk : __uint_as_float(1u));
                scale_ring[ring * 2 * kKeys + kKeys + t] = live ? rs[kPageTokens] : 0.0f;
                mbar_arrive(&tail->scale_full[ring]);
            }
            if (!wait_bar(&tail->empty[stage], ((u / L::kStages) & 1u) ^ 1u, failed)) return give_up(1 << 19);
            auto codes = [&](auto int8_t_) {
                constexpr bool kInt8 = decltype(int8_t_)::value;
                uint32_t src = src0 + slot * (kTileBytes / 2), to0 = dst0 + stage * kTileBytes, to1 = dst1 + stage * kTileBytes;
#pragma unroll 1
                for (int m = 0; m < kRows; m += 2) {
                    uint4 in[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(in[k].x), "=r"(in[k].y), "=r"(in[k].z), "=r"(in[k].w)
                                     : "r"(src + k * 4096));
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const uint32_t ws[4] = {in[k].x, in[k].y, in[k].z, in[k].w};
                        uint32_t h[8];
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            if constexpr (kInt8) u8x4_to_bf16(ws[w], h[2 * w], h[2 * w + 1]);
                            else e4m3x4_to_bf16(ws[w], h[2 * w], h[2 * w + 1]);
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to0 + k * 4096), "r"(h[0]), "r"(h[1]), "r"(h[2]),
                                     "r"(h[3])
                                     : "memory");
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to1 + k * 4096), "r"(h[4]), "r"(h[5]), "r"(h[6]),
                                     "r"(h[7])
                                     : "memory");
                    }
                    src += 8192;
                    to0 += 8192;
                    to1 += 8192;
                }
            };
            if (kv == 1 && p.v_int8) codes(std::true_type{});
            else codes(std::false_type{});
            mbar_arrive(&tail->raw_empty[slot]);
            fence_async_smem();
            mbar_arrive(&tail->full[stage]);
            ++u;
            return true;
        };
        while (ok && next_segment()) {
            const int n = s.t1 - s.t0;
            ok = item(s.t0, 0, tile_no);
            for (int i = 0; ok && i < n; ++i) {
                if (i + 1 < n) ok = item(s.t0 + i + 1, 0, tile_no + i + 1);
                ok = ok && item(s.t0 + i, 1, tile_no + i);
            }
            tile_no += n;
        }
    } else {
        set_regs_up<L::kSoftmaxRegs>();
        // ================= softmax and epilogue of lane l =================
        const int l = warp >> 2, quad = warp & 3, r = 32 * quad + lane;   // r: TMEM lane
        const uint32_t lane_addr = tmem + (static_cast<uint32_t>(32 * quad) << 16);
        const uint32_t tS = lane_addr + l * 128u, tO = lane_addr + kTmemO + l * 128u;
        uint32_t cnt = 0, tile_no = 0, seg_cnt = 0;   // tiles and segments of this lane
        // S of a tile is issued behind P V of the lane's previous one by the same thread, so s_full also says that O is
        // at rest and that the previous P has been read.
        auto wait = [&](uint64_t *bar, uint32_t par) {
            if (wait_bar(bar, par, failed)) return;
            if (!*failed) report_error(p.err, kErrWaitTimeout, kWhereChunkAttn, blockIdx.x, 1 << 22);
            *failed = 1;
        };

        auto rescale_o = [&](float alpha) {
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
        };

        // Rare: at chunk c (32 keys) of a tile, rows with `bad` take the largest score of the chunks from c on for their
        // reference; what they have so far, P of the earlier chunks included, is rescaled.
        auto outgrown = [&](int c, bool bad, bool unset, bool start, const float *ks, float &m_ref, float &l_run, float &tile_sum) {
            float top = -INFINITY;
#pragma unroll 1
            for (int k = c; k < 4; ++k) {
                uint32_t v[32];
                tmem_ld32_issue(tS + 32u * k, v);
                tmem_wait_ld32(v);
#pragma unroll
                for (int j = 0; j < 32; ++j) top = fmaxf(top, __uint_as_float(v[j]) * (k8 ? ks[32 * k + j] : p.scale_log2));
            }
            const float alpha = bad && !unset ? ex2_approx(m_ref - top) : 1.0f;
            if (bad) m_ref = top;
            l_run *= alpha;
            tile_sum *= alpha;
#pragma unroll 1
            for (int k = 0; k < c; ++k) {
                uint32_t v[16];
                tmem_ld_cols<16>(tS + 16u * k, v);
                tmem_wait_ld_regs<16>(v);
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = pack_bf16x2(bf16lo(v[j]) * alpha, bf16hi(v[j]) * alpha);
                tmem_st16(tS + 16u * k, v);
            }
            tmem_wait_st();
            if (!start) rescale_o(alpha);   // the first P V of a segment writes O anew
        };

        // Then P of the chunks [c, c1) by the new reference, over their S; their sums.  (Apart from the usual path: a
        // loop around that one, to go through it again, took 16 of the 186 us that ragged 8-bit segments needed then.)
        auto redo = [&](int c, int c1, const float *ks, const float *vs, float m_ref) -> float {
            const float sub = m_ref == -INFINITY ? 0.0f : m_ref;
            float sum = 0.0f;
#pragma unroll 1
            for (; c < c1; ++c) {
                uint32_t v[32], pk[16];
                tmem_ld32_issue(tS + 32u * c, v);
                tmem_wait_ld32(v);
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    float e[2];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        e[q] = ex2_approx(fmaf(__uint_as_float(v[j + q]), k8 ? ks[32 * c + j + q] : p.scale_log2, -sub));
                        sum += e[q];
                        if constexpr (k8) e[q] *= vs[32 * c + j + q];
                    }
                    pk[j / 2] = pack_bf16x2(e[0], e[1]);
                }
                tmem_st16(tS + 16u * c, pk);
            }
            return sum;
        };

        // Key tile kt (the ti-th of the segment) of pair and alternate mode; thread = query row.
        // No maximum is taken: the sums, which are needed anyway, tell when the reference will not do any more.
        auto row_tile = [&](int kt, int ti, bool masked, int pos, unsigned long long bits, bool start, float &m_ref, float &l_run,
                            float &want) {
            const uint32_t slot = (tile_no + ti) % L::kScaleRing;
            const float *ks = scale_ring + slot * 2 * kKeys, *vs = ks + kKeys;
            if constexpr (k8) wait(&tail->scale_full[slot], ((tile_no + ti) / L::kScaleRing) & 1u);
            if (__any_sync(0xffffffffu, want != m_ref)) {   // O is at rest (see s_full)
                const float alpha = want != m_ref ? ex2_approx(m_ref - want) : 1.0f;
                m_ref = want;
                l_run *= alpha;
                rescale_o(alpha);
            }
            if (masked) {
                // Scores of keys that the row does not see: -infinity, in place.  (The few tiles that need it share the
                // code of the rest.)
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const int k0 = kt * kKeys + 32 * c;
                    uint32_t seen;
                    if (!p.mask) {
                        const int d = pos - k0;
                        seen = d >= 31 ? 0xffffffffu : (d < 0 ? 0u : (2u << d) - 1u);
                    } else {
                        const int d = k0 - s.base;   // chunk token of the first key
                        seen = d <= -32 ? 0xffffffffu
                                        : (d < 0 ? ((1u << -d) - 1u) | static_cast<uint32_t>(bits << -d)
                                                 : (d < 64 ? static_cast<uint32_t>(bits >> d) : 0u));
                    }
                    if (__all_sync(0xffffffffu, seen == 0xffffffffu)) continue;
                    uint32_t v[32];
                    tmem_ld32_issue(tS + 32u * c, v);
                    tmem_wait_ld32(v);
                    float x[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = (seen >> j) & 1u ? __uint_as_float(v[j]) : -INFINITY;
                    tmem_st32(tS + 32u * c, x);
                }
                tmem_wait_st();
            }
            const uint64_t c2 = f2(p.scale_log2, p.scale_log2);
            float tile_sum = 0.0f;
            if constexpr (!k8) {
                uint32_t sr[2][32];
                tmem_ld32_issue(tS, sr[0]);
                // The whole tile unrolled, two chunks of S in registers, and P stored at its end, over S that is intact
                // until then: a 2048-row piece took 265 us when this was chosen, 320 with the short loop below.
                uint32_t pk[4][16];
#pragma unroll 1
                for (int again = 0; again < 2; ++again) {
                    const float sub = m_ref == -INFINITY ? 0.0f : m_ref;
                    const uint64_t nsub2 = f2(-sub, -sub);
                    uint64_t acc[2] = {f2(0.0f, 0.0f), f2(0.0f, 0.0f)};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        tmem_wait_ld32(sr[c & 1]);
                        if (c < 3) tmem_ld32_issue(tS + 32u * (c + 1), sr[(c + 1) & 1]);
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            float e[4];
                            un_f2(fma_f2(f2(__uint_as_float(sr[c & 1][j]), __uint_as_float(sr[c & 1][j + 1])), c2, nsub2), e[0], e[1]);
                            un_f2(fma_f2(f2(__uint_as_float(sr[c & 1][j + 2]), __uint_as_float(sr[c & 1][j + 3])), c2, nsub2), e[2], e[3]);
#pragma unroll
                            for (int q = 0; q < 4; ++q) e[q] = ex2_approx(e[q]);
                            acc[0] = add_f2(acc[0], f2(e[0], e[1]));
                            acc[1] = add_f2(acc[1], f2(e[2], e[3]));
                            pk[c][j / 2] = pack_bf16x2(e[0], e[1]);
                            pk[c][j / 2 + 1] = pack_bf16x2(e[2], e[3]);
                        }
                    }
                    float s0, s1;
                    un_f2(add_f2(acc[0], acc[1]), s0, s1);
                    tile_sum = s0 + s1;
                    const bool unset = m_ref == -INFINITY, bad = tile_sum > kSumMove || (unset && tile_sum < 1.0f / kSumMove);
                    if (!__any_sync(0xffffffffu, bad)) break;
                    if (again == 0) {
                        outgrown(0, bad, unset, start, ks, m_ref, l_run, tile_sum);
                        tmem_ld32_issue(tS, sr[0]);
                    }
                }
                if (m_ref == -INFINITY && tile_sum > 0.0f) m_ref = 0.0f;
                l_run += tile_sum;
                want = m_ref;
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_st16(tS + 16u * c, pk[c]);
                tmem_wait_st();
                return;
            }
            // The shortest code wins where the converting warps fetch theirs, too: ragged e4m3 segments take 155 us, 157 with
            // two chunks unrolled and 187 with the whole tile (158 and 188 against 153 with int8 V).
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                uint32_t sv[32], pk[16];
                tmem_ld32_issue(tS + 32u * c, sv);
                tmem_wait_ld32(sv);
                const float sub = m_ref == -INFINITY ? 0.0f : m_ref;
                const uint64_t nsub2 = f2(-sub, -sub);
                uint64_t acc[2] = {f2(0.0f, 0.0f), f2(0.0f, 0.0f)};
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 fk = *reinterpret_cast<const float4 *>(ks + 32 * c + j);
                    float e[4];
                    un_f2(fma_f2(f2(__uint_as_float(sv[j]), __uint_as_float(sv[j + 1])), f2(fk.x, fk.y), nsub2), e[0], e[1]);
                    un_f2(fma_f2(f2(__uint_as_float(sv[j + 2]), __uint_as_float(sv[j + 3])), f2(fk.z, fk.w), nsub2), e[2], e[3]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) e[q] = ex2_approx(e[q]);
                    acc[0] = add_f2(acc[0], f2(e[0], e[1]));
                    acc[1] = add_f2(acc[1], f2(e[2], e[3]));
                    const float4 fv = *reinterpret_cast<const float4 *>(vs + 32 * c + j);
                    un_f2(mul_f2(f2(e[0], e[1]), f2(fv.x, fv.y)), e[0], e[1]);
                    un_f2(mul_f2(f2(e[2], e[3]), f2(fv.z, fv.w)), e[2], e[3]);
                    pk[j / 2] = pack_bf16x2(e[0], e[1]);
                    pk[j / 2 + 1] = pack_bf16x2(e[2], e[3]);
                }
                float s0, s1;
                un_f2(add_f2(acc[0], acc[1]), s0, s1);
                float sum = s0 + s1;
                // Before P goes over S: has a term outgrown the range, or is a row's first sum too small to tell its
                // terms from zero (or has it none)?
                const bool unset = m_ref == -INFINITY, bad = sum > kSumMax || (unset && c == 0 && sum < 1.0f / kSumMax);
                if (__any_sync(0xffffffffu, bad)) {
                    outgrown(c, bad, unset, start, ks, m_ref, l_run, tile_sum);
                    sum = redo(c, c + 1, ks, vs, m_ref);
                } else {
                    tmem_st16(tS + 16u * c, pk);
                }
                if (m_ref == -INFINITY && sum > 0.0f) m_ref = 0.0f;
                tile_sum += sum;
            }
            l_run += tile_sum;
            // The range is wide; a row that leaves its middle moves its reference before the next tile.
            want = m_ref;
            if (tile_sum > kSumMove || (tile_sum < 1.0f / kSumMove && tile_sum > 0.0f && l_run == tile_sum))
                want += static_cast<float>((__float_as_int(tile_sum) >> 23) - 127);
            tmem_wait_st();
        };

        // A segment of thin mode: thread = key of a tile, then = output dim.  Columns n < 2 nq are row 2 i + h.
        auto thin_segment = [&](auto cols_t) {
            constexpr int kCols = decltype(cols_t)::value;
            const int n = s.t1 - s.t0, mine = lane_tiles(s, l);
            uint8_t *const sP = smem + kThinP + l * kThinPBytes;
            float *const ref = tail->thin_ref[l];
            float lsum[kCols];
#pragma unroll
            for (int j = 0; j < kCols; ++j) lsum[j] = 0.0f;
            for (int k = 0; k < mine; ++k) {
                const int ti = 2 * k + l, kt = s.t0 + ti, key = kt * kKeys + r;
                float kscale = p.scale_log2, vscale = 1.0f;
                if constexpr (k8) {
                    const uint32_t slot = (tile_no + ti) % L::kScaleRing;
                    wait(&tail->scale_full[slot], ((tile_no + ti) / L::kScaleRing) & 1u);
                    kscale = scale_ring[slot * 2 * kKeys + r];
                    vscale = scale_ring[slot * 2 * kKeys + kKeys + r];
                }
                wait(&tail->s_full[l], cnt & 1u);
                fence_after();
                uint32_t sr[kCols];
                tmem_ld_cols<kCols>(tS, sr);
                tmem_wait_ld_regs<kCols>(sr);
                float x[kCols];
#pragma unroll
                for (int j = 0; j < kCols; ++j) x[j] = __uint_as_float(sr[j]) * kscale;
                if (kt * kKeys + kKeys > s.q0pos) {     // the tile reaches the unit's queries
                    const int d = key - s.q0pos;        // this key among them (with a mask: among the chunk's tokens)
                    if (!p.mask) {
#pragma unroll
                        for (int j = 0; j < kCols; ++j) x[j] = (j >> 1) >= d ? x[j] : -INFINITY;
                    } else if (d >= 0) {
#pragma unroll
                        for (int j = 0; j < kCols; ++j) {
                            const bool see = j < 2 * s.nq && d < s.nq && ((__ldg(p.mask + s.row0 + (j >> 1)) >> d) & 1ull);
                            x[j] = see ? x[j] : -INFINITY;
                        }
                    }
                }
                bool move;
                if (k == 0) {
                    // References start from 0 if that serves: no score past 2^kRescaleLog2, and every column has one
                    // that is not far below.
                    uint32_t fair = 0;
                    float over = -INFINITY;
#pragma unroll
                    for (int j = 0; j < kCols; ++j) {
                        fair |= x[j] > -kRescaleLog2 ? 1u << j : 0u;
                        over = fmaxf(over, x[j]);
                    }
                    fair = __reduce_or_sync(0xffffffffu, fair);
                    if (__any_sync(0xffffffffu, over > kRescaleLog2)) fair = 0x80000000u;   // the mark for it
                    uint32_t *const words = reinterpret_cast<uint32_t *>(sP);
                    if (lane == 0) words[quad] = fair;
                    if (r < kCols) ref[r] = 0.0f;
                    bar_sync(kBarLane + l, 128);
                    const uint4 w = *reinterpret_cast<const uint4 *>(words);
                    constexpr uint32_t kAll = kCols == 32 ? 0xffffffffu : (1u << kCols % 32) - 1u;
                    const uint32_t every = w.x | w.y | w.z | w.w;
                    move = every != kAll || w.x == 0x80000000u || w.y == 0x80000000u || w.z == 0x80000000u || w.w == 0x80000000u;
                    bar_sync(kBarLane + l, 128);        // the scratch is read
                } else {
                    float over = -INFINITY;
#pragma unroll
                    for (int j = 0; j < kCols; ++j) over = fmaxf(over, x[j] - ref[j]);   // -inf - -inf: NaN, not the maximum
                    move = bar_any(kBarLane + l, 128, over > kRescaleLog2);
                }
                if (move) {
                    // New references: each column's maximum over the tile's keys, by warp, then over the four warps
                    // (scratch in the P tile).
                    float *const wmax = reinterpret_cast<float *>(sP);
#pragma unroll
                    for (int j = 0; j < kCols; ++j) {
                        const float m = warp_max(x[j]);
                        if (lane == 0) wmax[quad * kCols + j] = m;
                    }
                    bar_sync(kBarLane + l, 128);
                    float alpha[kCols];
#pragma unroll
                    for (int j = 0; j < kCols; ++j) {
                        const float m = fmaxf(fmaxf(wmax[j], wmax[kCols + j]), fmaxf(wmax[2 * kCols + j], wmax[3 * kCols + j]));
                        const float old = k > 0 ? ref[j] : -INFINITY;
                        alpha[j] = m > old ? ex2_approx(old - m) : 1.0f;
                        lsum[j] *= alpha[j];
                    }
                    bar_sync(kBarLane + l, 128);        // everyone has read the old references
                    if (r < kCols) {
                        const float m = fmaxf(fmaxf(wmax[r], wmax[kCols + r]), fmaxf(wmax[2 * kCols + r], wmax[3 * kCols + r]));
                        ref[r] = k > 0 ? fmaxf(ref[r], m) : m;
                    }
                    if (k > 0) {
                        fence_after();
                        uint32_t o[kCols];
                        tmem_ld_cols<kCols>(tO, o);
                        tmem_wait_ld_regs<kCols>(o);
                        if constexpr (kCols == 32) {
                            float f[32];
#pragma unroll
                            for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(o[j]) * alpha[j];
                            tmem_st32(tO, f);
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha[j]);
                            tmem_st16(tO, o);
                        }
                        tmem_wait_st();
                    }
                    bar_sync(kBarLane + l, 128);        // the references are written, the scratch is read
                }
                // P: this key's row of columns, swizzled in 16-byte chunks
                uint32_t pk[kCols / 2];
#pragma unroll
                for (int j = 0; j < kCols; j += 4) {
                    const float4 m = *reinterpret_cast<const float4 *>(ref + j);
                    const float ms[4] = {m.x, m.y, m.z, m.w};
                    float e[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        e[q] = ex2_approx(x[j + q] - (ms[q] == -INFINITY ? 0.0f : ms[q]));
                        lsum[j + q] += e[q];
                        if constexpr (k8) e[q] *= vscale;
                    }
                    pk[j / 2] = pack_bf16x2(e[0], e[1]);
                    pk[j / 2 + 1] = pack_bf16x2(e[2], e[3]);
                }
                const int turn = kCols == 16 ? (r >> 2) & 1 : (r >> 1) & 3;
#pragma unroll
                for (int c = 0; c < kCols / 8; ++c)
                    *reinterpret_cast<uint4 *>(sP + r * (2 * kCols) + ((c ^ turn) << 4)) =
                        make_uint4(pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
                fence_async_smem();
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&tail->p_full[l]);
                ++cnt;
            }
            if (mine > 0) {
                wait(&tail->o_full[l], seg_cnt++ & 1u);
                // Column sums over the lane's 128 threads.  (Not by way of the P tile: with the last P V done, the
                // loaders may already put a later segment's Q there.)
                float *const wsum = reinterpret_cast<float *>(&tail->ml[l][64]);
                warp_column_sums<kCols>(lsum, lane);
                if (lane % (32 / kCols) == 0) wsum[quad * kCols + lane / (32 / kCols)] = lsum[0];
                bar_sync(kBarLane + l, 128);
                if (r < kCols)
                    tail->ml[l][r] = make_float2(ref[r], (wsum[r] + wsum[kCols + r]) + (wsum[2 * kCols + r] + wsum[3 * kCols + r]));
            }
            fence_before();
            bar_sync(kBarBoth, 256);
            fence_after();
            // A column's factors for the lanes' O, by one thread each; the piece's (reference, sum) where it is one.
            const bool whole = s.first && s.last;
            const size_t piece = 2 * static_cast<size_t>(blockIdx.x) + (s.first ? 1 : 0);
            const int real = *failed ? 0 : 2 * s.nq;
            float2 *const factor = &tail->ml[0][32];
            if (l == 0 && r < kCols) {
                const float2 v0 = tail->ml[0][r], v1 = n > 1 ? tail->ml[1][r] : make_float2(-INFINITY, 0.0f);
                const float m = fmaxf(v0.x, v1.x);
                const float a0 = v0.y != 0.0f ? ex2_approx(v0.x - m) : 0.0f, a1 = v1.y != 0.0f ? ex2_approx(v1.x - m) : 0.0f;
                const float sum = a0 * v0.y + a1 * v1.y;
                const float norm = whole ? (sum != 0.0f ? 1.0f / sum : 0.0f) : 1.0f;
                factor[r] = make_float2(a0 * norm, a1 * norm);
                if (!whole && r < real) p.part_ml[piece * kPieceRows + r] = make_float2(m, sum);
            }
            bar_sync(kBarBoth, 256);
            // dims as threads: lane l finishes columns [l kCols / 2, (l + 1) kCols / 2), eight at a time
#pragma unroll 1
            for (int c = 0; c < kCols / 2; c += 8) {
                const int col0 = l * (kCols / 2) + c;
                uint32_t o0[8], o1[8];
                tmem_ld_cols<8>(lane_addr + kTmemO + col0, o0);
                tmem_ld_cols<8>(lane_addr + kTmemO + 128u + col0, o1);   // of a single tile's segment: not used
                tmem_wait_ld_regs<8>(o0);
                tmem_wait_ld_regs<8>(o1);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int col = col0 + j;
                    const float2 f = factor[col];
                    float o = f.x != 0.0f ? f.x * __uint_as_float(o0[j]) : 0.0f;
                    if (f.y != 0.0f) o += f.y * __uint_as_float(o1[j]);
                    if (col >= real) continue;
                    if (whole)
                        reinterpret_cast<__nv_bfloat16 *>(p.out)[static_cast<size_t>(s.row0 + (col >> 1)) * kQDim +
                                                                 (2 * s.g + (col & 1)) * kHeadDim + r] = __float2bfloat16_rn(o);
                    else
                        p.part_o[piece * (kPieceRows * kHeadDim) + col * kHeadDim + r] = o;
                }
            }
        };

        while (next_segment()) {
            const int n = s.t1 - s.t0;
            if (s.mode == kThin) {
                if (s.cols == 16) thin_segment(std::integral_constant<int, 16>{});
                else thin_segment(std::integral_constant<int, 32>{});
            } else {
                const int mine = lane_tiles(s, l), h = r & 1;
                const int qoff = s.pair() ? kQueries * l : 0;
                const int nq = min(kQueries, s.nq - qoff);
                const bool active = 32 * quad < 2 * nq;   // the warp holds a row of a query
                const int i = min(r >> 1, max(nq - 1, 0));
                const int pos_min = s.q0pos + qoff, pos = pos_min + i;
                unsigned long long bits = 0;
                if (p.mask && active) {
                    bits = p.mask[s.row0 + qoff + i];
                    if (s.nq < 64) bits &= (1ull << s.nq) - 1ull;
                }
                float m_ref = -INFINITY, l_run = 0.0f, want = -INFINITY;   // want: m_ref from the next tile on
                // tiles below `clear` are seen whole by every row
                const int step = s.pair() ? 1 : 2, ti0 = s.pair() ? 0 : l, clear = ((p.mask ? s.base : pos_min + 1) >> 7) - s.t0;
#pragma unroll 1
                for (int k = 0, ti = ti0; k < mine; ++k, ti += step) {
                    wait(&tail->s_full[l], cnt & 1u);
                    ++cnt;
                    fence_after();
                    if (active) row_tile(s.t0 + ti, ti, ti >= clear, pos, bits, k == 0, m_ref, l_run, want);
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&tail->p_full[l]);
                }
                if (mine > 0) wait(&tail->o_full[l], seg_cnt++ & 1u);
                const bool whole = s.first && s.last;
                float a0 = 1.0f, a1 = 0.0f, m_tot = m_ref, l_tot = l_run;
                if (!s.pair()) {
                    // Lane 1 says nothing for a single tile (and must not: lane 0 may still read its last entry).
                    if (mine > 0) tail->ml[l][r] = make_float2(m_ref, l_run);
                    fence_before();
                    bar_sync(kBarBoth, 256);
                    const float2 v0 = tail->ml[0][r], v1 = n > 1 ? tail->ml[1][r] : make_float2(-INFINITY, 0.0f);
                    m_tot = fmaxf(v0.x, v1.x);
                    a0 = v0.y != 0.0f ? ex2_approx(v0.x - m_tot) : 0.0f;
                    a1 = v1.y != 0.0f ? ex2_approx(v1.x - m_tot) : 0.0f;
                    l_tot = a0 * v0.y + a1 * v1.y;
                }
                fence_after();
                const bool real = r < 2 * nq && !*failed;
                if (active) {
                    const float norm = whole ? (l_tot != 0.0f ? 1.0f / l_tot : 0.0f) : 1.0f;
                    a0 *= norm;
                    a1 *= norm;
                    const int c0 = s.pair() ? 0 : 2 * l, c1 = s.pair() ? 4 : c0 + 2;   // 32-column chunks
                    const uint32_t o0 = s.pair() ? tO : lane_addr + kTmemO, o1 = lane_addr + kTmemO + 128u;
                    const bool own0 = s.pair() ? mine > 0 : true, two = !s.pair() && n > 1;
                    uint16_t *const out = p.out + static_cast<size_t>(s.row0 + qoff + i) * kQDim + (2 * s.g + h) * kHeadDim;
                    const size_t piece = 2 * static_cast<size_t>(blockIdx.x) + (s.first ? 1 : 0);
                    const int prow = (s.pair() ? 128 * l : 0) + r;
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
                    if (!whole && real && (s.pair() || l == 0))
                        p.part_ml[piece * kPieceRows + prow] = make_float2(m_tot, l_tot);
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tail->epi_done);
            if (!(s.first && s.last) && tid == 0)
                p.splits[2 * blockIdx.x + (s.first ? 1 : 0)] =
                    ChunkSplit{s.row0, s.nq, s.g, s.mode, s.c_first, s.c_last - s.c_first + 1};
            tile_no += n;
        }
    }
    fence_before();
    __syncthreads();
    if (warp == L::kLoadWarp && *failed) {   // no copy outlives the CTA: the last ones issued have landed
        constexpr uint32_t kRing = k8 ? L::kRaw : L::kStages;
        uint64_t *const ring_full = k8 ? tail->raw_full : tail->full;
        for (uint32_t k = 0; k < kRing; ++k) {
            const uint32_t item = tail->issued[k];
            if (item > 0) mbar_wait(&ring_full[k], ((item - 1) / kRing) & 1u, kWaitLimitCycles);
        }
        for (uint32_t q = tail->q_issued, k = 0; k < 2 && q > 0; ++k, --q)
            mbar_wait(&tail->q_full[(q - 1) & 1u], ((q - 1) >> 1) & 1u, kWaitLimitCycles);
    }
    if (warp == kMmaWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// Joins the pieces of the units that are cut: o = sum_p 2^(m_p - M) o_p /
// sum_p 2^(m_p - M) l_p, pieces in order.  As many blocks (times gridDim.y) share
// a unit as it has pieces: those of the CTAs that held one, which are two units'
// at most.  Thread = (row, four dims), in the order the pieces lie in memory:
// thin mode's row by row, the others' four dims of all rows together.  Bound by
// the latency of a launch and its dependent loads; kJoinBatch pieces' are in
// flight together.  When that was one piece at a time by the first CTA's blocks
// alone, 100 rows on 3000 tokens (some 20 pieces a unit) took 47 us instead of
// 20, 5 rows on 512 tokens 11.2 us instead of 10.1.  More or larger blocks cost the small
// launch what they give the large one.
constexpr int kJoinThreads = 128, kJoinBatch = 6, kJoinRows = 8;

__global__ void __launch_bounds__(kJoinThreads) chunk_join_kernel(const __grid_constant__ ChunkAttendParams p) {
    pdl_trigger();
    pdl_wait();
    const ChunkSplit both[2] = {p.splits[2 * blockIdx.x], p.splits[2 * blockIdx.x + 1]};
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
        const ChunkSplit d = side ? both[1] : both[0];
        const int c0 = d.c_first, c_last = c0 + d.n - 1, rows = 2 * d.nq;   // pair: lane 0's 128 rows, then lane 1's
        if (d.n < 2) continue;
        for (int w = ((blockIdx.x - c0) * gridDim.y + blockIdx.y) * kJoinThreads + threadIdx.x; w < rows * (kHeadDim / 4);
             w += d.n * gridDim.y * kJoinThreads) {
            const bool thin = d.mode == kThin;
            const int r = thin ? w / (kHeadDim / 4) : w % rows, c = thin ? w % (kHeadDim / 4) : w / rows;
            const size_t off = thin ? static_cast<size_t>(w) * 4 : static_cast<size_t>(c) * (kPieceRows * 4) + r * 4;
            float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int k = c0; k <= c_last; k += kJoinBatch) {
                float2 ml[kJoinBatch];
                float4 v[kJoinBatch];
#pragma unroll
                for (int b = 0; b < kJoinBatch; ++b) {
                    ml[b] = make_float2(-INFINITY, 0.0f);
                    v[b] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (k + b > c_last) continue;
                    const size_t piece = 2 * (k + b) + (k + b == c0 ? 1 : 0);
                    ml[b] = p.part_ml[piece * kPieceRows + r];
                    v[b] = *reinterpret_cast<const float4 *>(p.part_o + piece * (kPieceRows * kHeadDim) + off);
                }
                float top = m;
#pragma unroll
                for (int b = 0; b < kJoinBatch; ++b) top = ml[b].y > 0.0f ? fmaxf(top, ml[b].x) : top;
                const float keep = l != 0.0f ? exp2f(m - top) : 0.0f;
                m = top;
                l *= keep;
#pragma unroll
                for (int q = 0; q < 4; ++q) o[q] *= keep;
#pragma unroll
                for (int b = 0; b < kJoinBatch; ++b) {
                    if (ml[b].y == 0.0f) continue;   // (a piece that saw nothing of the row)
                    const float a = exp2f(ml[b].x - m);
                    l += a * ml[b].y;
                    o[0] += a * v[b].x;
                    o[1] += a * v[b].y;
                    o[2] += a * v[b].z;
                    o[3] += a * v[b].w;
                }
            }
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            uint16_t *out = p.out + static_cast<size_t>(d.row0 + (r >> 1)) * kQDim + (2 * d.g + (r & 1)) * kHeadDim + 4 * c;
            *reinterpret_cast<uint2 *>(out) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
        }
    }
}

template <bool k8> size_t smem_want() { return Layout<k8>::kTailOff + sizeof(Tail) + 1023; }

size_t smem_capped(size_t want, int optin) { return want < static_cast<size_t>(optin) ? want : static_cast<size_t>(optin); }

cudaError_t smem_optin(int *optin) {
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    return e != cudaSuccess ? e : cudaDeviceGetAttribute(optin, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

bool encode_3d(CUtensorMap *m, CUtensorMapDataType type, const void *ptr, const cuuint64_t (&dims)[3],
               const cuuint64_t (&strides)[2], const cuuint32_t (&box)[3], CUtensorMapSwizzle swizzle) {
    const auto enc = reinterpret_cast<EncodeTiled>(tensor_map_encoder());
    const cuuint32_t step[3] = {1, 1, 1};
    return enc && enc(m, type, 3, const_cast<void *>(ptr), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool encode_maps(Maps *m, const ChunkAttendParams &p, bool k8) {
    const cuuint64_t elem = k8 ? 1 : 2, page_rows = 2 * kHkv * kPageTokens;
    const cuuint64_t kv_dims[3] = {kHeadDim, page_rows, static_cast<cuuint64_t>(p.n_pages)};
    const cuuint64_t kv_strides[2] = {kHeadDim * elem, kHeadDim * elem * page_rows};
    const cuuint32_t kv_box[3] = {k8 ? 128u : 64u, kPageTokens, 1};
    const cuuint64_t q_dims[3] = {kHeadDim, kHq, static_cast<cuuint64_t>(p.rows)};
    const cuuint64_t q_strides[2] = {kHeadDim * 2, kQDim * 2};
    const cuuint32_t q_box[3] = {64, kHq / kHkv, kQueries}, thin_box[3] = {64, kHq / kHkv, kThinQueries};
    if (k8) {
        const auto enc = reinterpret_cast<EncodeTiled>(tensor_map_encoder());
        const cuuint64_t dims[4] = {kPageTokens, kHkv, 2, static_cast<cuuint64_t>(p.n_pages)};
        const cuuint64_t strides[3] = {kPageTokens * 4, kHkv * kPageTokens * 4, 2 * kHkv * kPageTokens * 4};
        const cuuint32_t box[4] = {kPageTokens, 1, 2, 1}, step[4] = {1, 1, 1, 1};
        if (!enc || enc(&m->scales, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, const_cast<float *>(p.scales), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    }
    return encode_3d(&m->kv, k8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.pool, kv_dims, kv_strides,
                     kv_box, CU_TENSOR_MAP_SWIZZLE_128B) &&
           encode_3d(&m->q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.q, q_dims, q_strides, q_box, CU_TENSOR_MAP_SWIZZLE_128B) &&
           encode_3d(&m->q_thin, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.q, q_dims, q_strides, thin_box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool k8> cudaError_t launch_main(const ChunkAttendParams &p, int num_sms, cudaStream_t st) {
    int optin = 0;
    const cudaError_t e = smem_optin(&optin);
    if (e != cudaSuccess) return e;
    Maps maps{};
    if (!encode_maps(&maps, p, k8)) return cudaErrorInvalidValue;
    return launch_pdl(chunk_attn_kernel<k8>, dim3(num_sms), dim3(Layout<k8>::kThreads), smem_capped(smem_want<k8>(), optin), st, p,
                      maps);
}

}  // namespace

// Whether the work of a call, counted as the kernel does, stays below 2^31 whatever its lists say.
bool chunk_work_fits(int n, int rows, int maxp) {
    const long long blocks = rows / (2 * kQueries) + static_cast<long long>(n);
    const long long tiles = (static_cast<long long>(maxp) * kPageTokens + kKeys - 1) / kKeys;
    return blocks * (2 * tiles + kPairUnitCost) * kHkv < 1ll << 31;
}

ChunkWorkspace chunk_workspace(int num_sms) {
    const size_t pieces = 2 * static_cast<size_t>(num_sms);
    return ChunkWorkspace{pieces * kPieceRows * kHeadDim, pieces * kPieceRows, pieces};
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
    cudaError_t e = cudaErrorInvalidValue;
    if (kv_dtype == kKvBF16) e = launch_main<false>(p, num_sms, st);
    else if (kv_is_8bit(kv_dtype)) e = launch_main<true>(p, num_sms, st);
    if (e != cudaSuccess) return e;
    return launch_pdl(chunk_join_kernel, dim3(num_sms, kJoinRows), dim3(kJoinThreads), 0, st, p);
}

}  // namespace qkv
