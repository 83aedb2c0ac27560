// Chunk attention: the entry points, and the merge of split partials.
#include "kush_attend.cuh"

namespace kush {

// One warp per (row, q head): o = sum_z e^(m_z - M) o_z / sum_z e^(m_z - M) l_z, lane z % 32 holding the factors of its splits,
// the partial outputs read D/32 channels a lane.  The arithmetic is merge_splits' (sums in split order, fmaf, one division), so
// that the windowed decode's output does not depend on which merge it takes.  Rows before the first sequence and behind the last
// one (before qsl[0], from qsl[S] on; qsl null: none) have no partials and are left as they are.
template <int D, class IN>
__global__ void __launch_bounds__(128) chunk_combine_kernel(IN* __restrict__ out, const float* __restrict__ part_ml,
                                                            const float* __restrict__ part_o, int n_splits, int H, int G,
                                                            const int32_t* __restrict__ qsl, int S, int64_t units) {
    constexpr int R = D / WARP;
    pdl_wait();
    const int lane = threadIdx.x % WARP;
    const int64_t u = int64_t(blockIdx.x) * 4 + threadIdx.x / WARP;           // (row * H + h) * G + g
    if (u >= units) return;
    if (const int64_t row = u / (H * G); qsl && (row < qsl[0] || row >= qsl[S])) return;
    const int64_t first = (u / G) * n_splits * G + u % G;                    // its partial of split 0; split z at + z G
    float M = -INFINITY;
    for (int z = lane; z < n_splits; z += WARP) M = fmaxf(M, part_ml[2 * (first + int64_t(z) * G)]);
    M = warp_max(M);
    float L = 0.0f, o[R];
#pragma unroll
    for (int i = 0; i < R; i++) o[i] = 0.0f;
    for (int z0 = 0; z0 < n_splits; z0 += WARP) {
        float f = 0.0f, l = 0.0f;
        bool part = false;                                                    // an empty split's partial output is not written
        if (z0 + lane < n_splits) {
            const float2 ml = *reinterpret_cast<const float2*>(part_ml + 2 * (first + int64_t(z0 + lane) * G));
            part = ml.x > -INFINITY;
            if (part) {
                f = __expf(ml.x - M);
                l = ml.y;
            }
        }
        const unsigned parts = __ballot_sync(0xffffffffu, part);
        const int nz = min(WARP, n_splits - z0);
        for (int z = 0; z < nz; z++) {
            if (!(parts >> z & 1u)) continue;
            const float fz = __shfl_sync(0xffffffffu, f, z);
            L = fmaf(__shfl_sync(0xffffffffu, l, z), fz, L);
            const float* po = part_o + (first + int64_t(z0 + z) * G) * D + lane * R;
            float v[R];
            if constexpr (R == 2) {
                *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(po);
            } else {
#pragma unroll
                for (int i = 0; i < R; i += 4) *reinterpret_cast<float4*>(v + i) = *reinterpret_cast<const float4*>(po + i);
            }
#pragma unroll
            for (int i = 0; i < R; i++) o[i] = fmaf(fz, v[i], o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++) out[u * D + lane * R + i] = from_f32<IN>(L > 0.0f ? o[i] / L : L);      // (0, or a NaN that came with a partial)
}

int launch_chunk_combine(int D, int dtype, const AttendArgs& a, int64_t rows, cudaStream_t stream) {
    const int64_t units = rows * a.H * a.G, blocks = (units + 3) / 4;
    if (blocks > 0x7fffffff) return set_error(KUSH_ERR_ARG, "attention: %lld rows to merge", (long long)rows);
    return dispatch_dim(D, [&](auto Dc) {
        return dispatch_dtype(dtype, [&](auto in) {
            using IN = decltype(in);
            launch_pdl(chunk_combine_kernel<Dc.value, IN>, dim3(unsigned(blocks)), dim3(128), 0, stream,
                       static_cast<IN*>(a.out), const_cast<const float*>(a.part_ml), const_cast<const float*>(a.part_o),
                       int(a.n_splits), int(a.H), int(a.G), a.qsl, int(a.S), units);
            return check_launch("attention (combine)");
        });
    });
}

}  // namespace kush

using namespace kush;

static int attend_chunk(int32_t head_dim, int32_t bits, int32_t page, int32_t dtype, int32_t group, const void* q, int64_t q_stride,
                        const void* k_new, const void* v_new, int64_t k_stride, int64_t v_stride, void* out,
                        const int32_t* query_start_loc, const int32_t* seq_lens, const int32_t* tail_idx, const void* cache,
                        int64_t block_stride, int64_t head_stride, const void* tail_k, const int32_t* block_table,
                        int64_t max_pages, int32_t hkv, float scale, int32_t window, int32_t sinks, int32_t n_splits,
                        float* part_ml, float* part_o, int64_t n_rows, int32_t n_seqs, void* stream, int32_t held_slot = 0,
                        int32_t held_tile = 0, int32_t limit_ms = 0) {
    static const char* what = "kush_sm100_attend_chunk";
    if (kush_sm100_record_bytes(head_dim, bits, page) == 0 || dtype < KUSH_F16 || dtype > KUSH_F32)
        return set_error(KUSH_ERR_UNSUPPORTED, "%s: unsupported head_dim %d / bits %d / page %d / dtype %d", what, head_dim,
                         bits, page, dtype);
    if (n_rows < 0 || n_seqs < 0 || hkv < 1 || group < 1 || n_splits < 1 || window < 0 || sinks < 0)
        return set_error(KUSH_ERR_ARG, "%s: n_rows %lld n_seqs %d hkv %d group %d n_splits %d window %d sinks %d", what,
                         (long long)n_rows, n_seqs, hkv, group, n_splits, window, sinks);
    if (n_rows == 0 || n_seqs == 0) return KUSH_OK;
    if (!q || !k_new || !v_new || !out || !query_start_loc || !seq_lens || !tail_idx || !cache || !tail_k || !block_table)
        return set_error(KUSH_ERR_ARG, "%s: null pointer", what);
    if (n_splits > 1 && (!part_ml || !part_o))
        return set_error(KUSH_ERR_ARG, "%s: n_splits %d needs part_ml and part_o", what, n_splits);
    if (n_rows * group > 0x7fffffff)
        return set_error(KUSH_ERR_ARG, "%s: %lld rows of %d q heads per kv head", what, (long long)n_rows, group);
    const int64_t size = dtype == KUSH_F32 ? 4 : 2;
    if (!aligned16(cache) || (block_stride & 15) || (head_stride & 15))
        return set_error(KUSH_ERR_ARG, "%s: records must be 16-byte aligned (cache %p, strides %lld %lld)", what, cache,
                         (long long)block_stride, (long long)head_stride);
    if (!aligned16(q) || !aligned16(k_new) || !aligned16(v_new) || !aligned16(out) || !aligned16(tail_k) ||
        ((q_stride * size) & 15) || ((k_stride * size) & 15) || ((v_stride * size) & 15))
        return set_error(KUSH_ERR_ARG, "%s: rows of q, k, v, out and tail_k must be 16-byte aligned", what);
    if (n_splits > 1 && (!aligned16(part_o) || (reinterpret_cast<uintptr_t>(part_ml) & 7)))
        return set_error(KUSH_ERR_ARG, "%s: part_ml must be 8-byte and part_o 16-byte aligned", what);
    AttendArgs a{};
    a.q = q;
    a.out = out;
    a.k_new = k_new;
    a.v_new = v_new;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.cache = static_cast<const uint8_t*>(cache);
    a.block_stride = block_stride;
    a.head_stride = head_stride;
    a.tail_k = tail_k;
    a.tail_idx = tail_idx;
    a.block_table = block_table;
    a.seq_lens = seq_lens;
    a.qsl = query_start_loc;
    a.max_pages = max_pages;
    a.H = hkv;
    a.G = group;
    a.S = n_seqs;
    a.n_rows = int32_t(n_rows);
    a.sm_log2 = scale * 1.4426950408889634f;
    a.window = window < KUSH_NO_POSITION ? window : KUSH_NO_POSITION;     // (differences of positions stay in 32 bits)
    a.sinks = sinks < KUSH_NO_POSITION ? sinks : KUSH_NO_POSITION;
    a.n_splits = n_splits;
    a.part_ml = part_ml;
    a.part_o = part_o;
    a.held = {held_slot, held_tile, limit_ms};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rc = attend_tc_supported(head_dim, dtype) ? launch_attend_tc(head_dim, bits, page, dtype, a, n_rows, st)
                                                        : launch_attend_simt(head_dim, bits, page, dtype, a, n_rows, st);
    if (rc != KUSH_OK || n_splits == 1) return rc;
    return launch_chunk_combine(head_dim, dtype, a, n_rows, st);
}

extern "C" int kush_sm100_attend_chunk(int32_t head_dim, int32_t bits, int32_t page, int32_t dtype, int32_t group,
                                       const void* q, int64_t q_stride, const void* k_new, const void* v_new,
                                       int64_t k_stride, int64_t v_stride, void* out, const int32_t* query_start_loc,
                                       const int32_t* seq_lens, const int32_t* tail_idx, const void* cache,
                                       int64_t block_stride, int64_t head_stride, const void* tail_k,
                                       const int32_t* block_table, int64_t max_pages, int32_t hkv, float scale,
                                       int32_t window, int32_t sinks, int32_t n_splits, float* part_ml, float* part_o,
                                       int64_t n_rows, int32_t n_seqs, void* stream) {
    return attend_chunk(head_dim, bits, page, dtype, group, q, q_stride, k_new, v_new, k_stride, v_stride, out,
                        query_start_loc, seq_lens, tail_idx, cache, block_stride, head_stride, tail_k, block_table, max_pages, hkv, scale, window, sinks,
                        n_splits, part_ml, part_o, n_rows, n_seqs, stream);
}

extern "C" int kush_sm100_attend_chunk_held(int32_t head_dim, int32_t bits, int32_t page, int32_t dtype, int32_t group,
                                            const void* q, int64_t q_stride, const void* k_new, const void* v_new,
                                            int64_t k_stride, int64_t v_stride, void* out, const int32_t* query_start_loc,
                                            const int32_t* seq_lens, const int32_t* tail_idx, const void* cache,
                                            int64_t block_stride, int64_t head_stride, const void* tail_k,
                                            const int32_t* block_table, int64_t max_pages, int32_t hkv, float scale,
                                            int32_t window, int32_t sinks, int32_t n_splits, float* part_ml, float* part_o,
                                            int64_t n_rows, int32_t n_seqs, int32_t held_slot, int32_t held_tile,
                                            int32_t limit_ms, void* stream) {
    if (held_slot < 0 || held_slot > 1 || held_tile < 0 || limit_ms < 1 || limit_ms > 2000)
        return set_error(KUSH_ERR_ARG, "kush_sm100_attend_chunk_held: slot %d tile %d limit_ms %d", held_slot, held_tile, limit_ms);
    if (head_dim != 128 || bits != 4 || page != 16 || dtype != KUSH_BF16)
        return set_error(KUSH_ERR_UNSUPPORTED, "kush_sm100_attend_chunk_held: head_dim 128, 4 bits, pages of 16, bf16 only");
    return attend_chunk(head_dim, bits, page, dtype, group, q, q_stride, k_new, v_new, k_stride, v_stride, out,
                        query_start_loc, seq_lens, tail_idx, cache, block_stride, head_stride, tail_k, block_table, max_pages, hkv, scale, window, sinks,
                        n_splits, part_ml, part_o, n_rows, n_seqs, stream, held_slot, held_tile, limit_ms);
}
