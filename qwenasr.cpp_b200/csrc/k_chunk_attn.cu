// Attention of a chunk of new tokens of each stream over its pages: the chunk's
// queries see the tokens before the chunk and, inside it, the tokens up to
// their own (or those of a draft-tree mask).
//
// out[r] = sum_k softmax_k(q_r . k / sqrt(128)) v over the visible tokens; zero
// where none is visible.
#include "kernels.h"

namespace qkv {

namespace {

// One warp per (row, head), a lane four dims, one token at a time.
template <typename TC>
__global__ void __launch_bounds__(kHq * 32) chunk_attn_kernel(ChunkAttendParams p) {
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.x, head = threadIdx.x >> 5, lane = threadIdx.x & 31, g = head / (kHq / kHkv);
    // The last stream that starts at or before the row (later empty chunks share its start).
    int lo = 0, hi = p.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.starts[mid] <= row) lo = mid;
        else hi = mid;
    }
    while (lo > 0 && p.starts[lo + 1] <= row) --lo;
    const int i = lo;
    bool before = false;   // an earlier entry ends behind this one's start
    for (int j = threadIdx.x; j < p.n; j += blockDim.x) {
        if (j < i && p.starts[j + 1] > p.starts[i]) before = true;
        if (row == 0 && p.slots[j] != -1 && (p.starts[j] < 0 || p.starts[j + 1] < p.starts[j] || p.starts[j + 1] > p.rows))
            report_error(p.err, kErrRowBounds, kWhereChunkAttn, j, p.starts[j]);
    }
    before = __syncthreads_or(before);
    const int first = p.starts[i], m = p.starts[i + 1] - first, len = p.lens[i], slot = p.slots[i];
    if (row < first || row >= first + m || slot == -1) return;   // behind the last chunk, or padding
    const bool ok = !before && slot >= 0 && slot < p.max_streams && first >= 0 && first + m <= p.rows && len >= m &&
                    (len + kPageTokens - 1) / kPageTokens <= p.maxp && (!p.mask || m <= 64);
    if (!ok) {
        if (threadIdx.x == 0) report_error(p.err, kErrRowBounds, kWhereChunkAttn, i, len);
        return;
    }
    const int base = len - m;
    const unsigned long long bits = p.mask ? p.mask[row] : 0;
    const int end = p.mask ? len : base + (row - first) + 1;
    const size_t q_off = static_cast<size_t>(row) * kQDim + head * kHeadDim + 4 * lane;
    const uint2 qw = *reinterpret_cast<const uint2 *>(p.q + q_off);
    const float q[4] = {bf16lo(qw.x), bf16hi(qw.x), bf16lo(qw.y), bf16hi(qw.y)};
    const int *pt = p.page_table + static_cast<size_t>(slot) * p.maxp;
    float m_run = -INFINITY, l_run = 0.0f, o[4] = {};
    for (int t = 0; t < end; ++t) {
        if (p.mask && t >= base && !((bits >> (t - base)) & 1)) continue;
        const int page = pt[t / kPageTokens];
        if (page < 0 || page >= p.n_pages) {
            if (threadIdx.x == 0) report_error(p.err, kErrPageIndex, kWhereChunkAttn, i, page);
            return;
        }
        const size_t kvec = ((static_cast<size_t>(page) * 2) * kHkv + g) * kPageTokens + t % kPageTokens;
        const size_t vvec = kvec + static_cast<size_t>(kHkv) * kPageTokens;
        float k[4], v[4];
        if constexpr (sizeof(TC) == 2) {
            const uint2 kw = reinterpret_cast<const uint2 *>(p.pool)[kvec * 32 + lane];
            const uint2 vw = reinterpret_cast<const uint2 *>(p.pool)[vvec * 32 + lane];
            k[0] = bf16lo(kw.x), k[1] = bf16hi(kw.x), k[2] = bf16lo(kw.y), k[3] = bf16hi(kw.y);
            v[0] = bf16lo(vw.x), v[1] = bf16hi(vw.x), v[2] = bf16lo(vw.y), v[3] = bf16hi(vw.y);
        } else {
            const uint32_t kw = reinterpret_cast<const uint32_t *>(p.pool)[kvec * 32 + lane];
            const uint32_t vw = reinterpret_cast<const uint32_t *>(p.pool)[vvec * 32 + lane];
            const float ks = p.scales[kvec], vs = p.scales[vvec];
            const float2 k01 = e4m3x2_to_f2(static_cast<uint16_t>(kw)), k23 = e4m3x2_to_f2(static_cast<uint16_t>(kw >> 16));
            k[0] = k01.x * ks, k[1] = k01.y * ks, k[2] = k23.x * ks, k[3] = k23.y * ks;
            if (p.v_int8) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = u8ex_to_f((vw >> (8 * j)) & 0xffu) * vs;
            } else {
                const float2 v01 = e4m3x2_to_f2(static_cast<uint16_t>(vw)), v23 = e4m3x2_to_f2(static_cast<uint16_t>(vw >> 16));
                v[0] = v01.x * vs, v[1] = v01.y * vs, v[2] = v23.x * vs, v[3] = v23.y * vs;
            }
        }
        float s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= p.scale_log2;
        const float m_new = fmaxf(m_run, s);
        const float alpha = exp2f(m_run - m_new), e = exp2f(s - m_new);
        m_run = m_new;
        l_run = l_run * alpha + e;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = o[j] * alpha + e * v[j];
    }
    const float inv = l_run > 0.0f ? 1.0f / l_run : 0.0f;
    *reinterpret_cast<uint2 *>(p.out + q_off) =
        make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
}

}  // namespace

cudaError_t launch_chunk_attn(const ChunkAttendParams &p, int kv_dtype, cudaStream_t st) {
    if (p.n <= 0 || p.rows <= 0) return cudaSuccess;
    if (kv_dtype == kKvBF16)
        return launch_pdl(chunk_attn_kernel<__nv_bfloat16>, dim3(p.rows), dim3(kHq * 32), 0, st, p);
    if (kv_is_8bit(kv_dtype))
        return launch_pdl(chunk_attn_kernel<uint8_t>, dim3(p.rows), dim3(kHq * 32), 0, st, p);
    return cudaErrorInvalidValue;
}

}  // namespace qkv
