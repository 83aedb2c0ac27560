// Chunk attention, and the windowed decode, on the CUDA cores in fp32: the configurations the tensor-core kernels do not
// take (fp32 rows, head_dim 256 in the chunk form, large GQA groups in the windowed decode).
//
// A block of 128 threads holds a tile of 32 query rows and walks the key tiles of 32 tokens it sees: keys and values are
// dequantized into shared memory (c * s + b in fp32; tail and new rows as they are; tokens that no row of the tile sees
// are zeros and neither they nor their pages are read), scores in a 4 x 2 register tile per thread, an online softmax
// with running maximum and sum per row, then the 4 x D/16 register tile of the output.  Bound by fp32 FMAs and the
// shared-memory loads that feed them: 2 sequences x 100 rows of 32 q heads over 2000
// int4 tokens in fp32 take 434 us = 15.5 TFLOP/s; a decoded token's rows (fewer than the tile's 32) are bound by the tiles'
// loads, four tokens of a warp in flight (one sequence, window 8192, 51 splits: 108 us).
#include "kush_attend.cuh"

namespace kush {

constexpr int AS_TM = 32, AS_TN = 32, AS_THREADS = 128;

template <int D>
struct AsSmem {
    static constexpr int QP = D + 4;                       // padded row pitches (floats): conflict-free float4 columns
    static constexpr int Q = AS_TM * QP, K = AS_TN * QP, V = AS_TN * D, SC = AS_TM * (AS_TN + 1);
    static constexpr int BYTES = 4 * (Q + K + V + SC + 3 * AS_TM);
};

template <int D, int BITS, int P, class IN>
__global__ void __launch_bounds__(AS_THREADS) attend_simt_kernel(AttendArgs a) {
    using F = Fmt<D, BITS, P>;
    using M = AsSmem<D>;
    constexpr int QP = M::QP, SP = AS_TN + 1, R = D / WARP, DV = D / 64;     // DV: float4 of output dims per thread
    extern __shared__ float4 smem4[];
    float* qs = reinterpret_cast<float*>(smem4);           // [TM][QP] q * scale * log2 e
    float* ks = qs + M::Q;                                 // [TN][QP]
    float* vs = ks + M::K;                                 // [TN][D]
    float* sc = vs + M::V;                                 // [TM][SP] scores, then weights
    float *mrow = sc + M::SC, *lrow = mrow + AS_TM, *crow = lrow + AS_TM;
    pdl_wait();
    const int h = blockIdx.y, z = blockIdx.z, tid = threadIdx.x, wid = tid / WARP, lane = tid % WARP;
    RowTile t;
    if (!row_tile(a, a.qsl ? int(gridDim.x) - 1 - int(blockIdx.x) : int(blockIdx.x), AS_TM, t)) return;
    const KeyTiles kt = key_tiles(t.p0, t.p1, a.window, a.sinks, AS_TN);
    int i0, i1;
    key_split(a, z, AS_TM, AS_TN, kt.count, i0, i1);
    auto grow = [&](int r) { return t.q0 + (t.r0 + r) / a.G; };              // global row and q head of tile row r
    auto head = [&](int r) { return h * a.G + (t.r0 + r) % a.G; };
    if (a.n_splits > 1 && i0 >= i1) {                                        // nothing here: empty partials
        for (int r = tid; r < t.nr; r += AS_THREADS) {
            float* ml = a.part_ml + 2 * part_row(a, grow(r), h, z, (t.r0 + r) % a.G);
            ml[0] = -INFINITY;
            ml[1] = 0.0f;
        }
        return;
    }
    const IN* q = static_cast<const IN*>(a.q);
    for (int i = tid; i < AS_TM * D; i += AS_THREADS) {
        const int r = i / D, d = i % D;
        qs[r * QP + d] = r < t.nr ? to_f32(q[grow(r) * a.q_stride + int64_t(head(r)) * D + d]) * (a.rot ? 1.0f : a.sm_log2) : 0.0f;
    }
    if (a.rot) {
        __syncthreads();
        for (int r = wid; r < t.nr; r += AS_THREADS / WARP) {
            float x[R];
#pragma unroll
            for (int i = 0; i < R; i++) x[i] = qs[r * QP + lane + WARP * i];
            fwht_warp<D>(x, lane);
#pragma unroll
            for (int i = 0; i < R; i++) qs[r * QP + lane + WARP * i] = x[i] * a.sm_log2;
        }
    }
    for (int r = tid; r < AS_TM; r += AS_THREADS) {
        mrow[r] = -INFINITY;
        lrow[r] = 0.0f;
    }
    const int ty = tid / 16, tx = tid % 16;                // rows 4 ty .. + 3; score columns tx, tx + 16; dims 4 tx + 64 i
    float4 acc[4][DV];
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
        for (int i = 0; i < DV; i++) acc[r][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int32_t* bt = a.block_table + int64_t(t.s) * a.max_pages;
    const IN* tail = static_cast<const IN*>(a.tail_k) + (int64_t(a.tail_idx[t.s]) * a.H + h) * P * D;
    const int full = t.ctx / P * P;                        // cached tokens in finished pages
    for (int it = i0; it < i1; it++) {
        const int j0 = kt.tile(it) * AS_TN;
        __syncthreads();
        // a warp per token, lanes over channels, four tokens' loads in flight
#pragma unroll 1
        for (int c0 = wid; c0 < AS_TN; c0 += 4 * (AS_THREADS / WARP)) {
            float kx[4][R], vx[4][R];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int j = j0 + c0 + u * (AS_THREADS / WARP);
#pragma unroll
                for (int i = 0; i < R; i++) kx[u][i] = vx[u][i] = 0.0f;
                if (!kt.seen(j, t.p1)) continue;
                if (j < t.ctx) {
                    const uint8_t* rec = a.cache + int64_t(bt[j / P]) * a.block_stride + int64_t(h) * a.head_stride;
                    const int s = j % P;
                    const float vsc = h_load(rec + F::OFF_VS, s), vbi = h_load(rec + F::OFF_VB, s);
#pragma unroll
                    for (int i = 0; i < R; i++) {
                        const int d = lane + WARP * i;
                        kx[u][i] = j < full ? fmaf(float(code_at<D, BITS>(rec + s * F::DC, d)), h_load(rec + F::OFF_KS, d),
                                                   h_load(rec + F::OFF_KB, d))
                                            : to_f32(tail[s * D + d]);
                        vx[u][i] = fmaf(float(code_at<D, BITS>(rec + F::OFF_VQ + s * F::DC, d)), vsc, vbi);
                    }
                } else {
                    const int64_t row = t.q0 + (j - t.ctx);
                    const IN* kn = static_cast<const IN*>(a.k_new) + row * a.k_stride + int64_t(h) * D;
                    const IN* vn = static_cast<const IN*>(a.v_new) + row * a.v_stride + int64_t(h) * D;
#pragma unroll
                    for (int i = 0; i < R; i++) {
                        kx[u][i] = to_f32(kn[lane + WARP * i]);
                        vx[u][i] = to_f32(vn[lane + WARP * i]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int c = c0 + u * (AS_THREADS / WARP);
#pragma unroll
                for (int i = 0; i < R; i++) {
                    ks[c * QP + lane + WARP * i] = kx[u][i];
                    vs[c * D + lane + WARP * i] = vx[u][i];
                }
            }
        }
        __syncthreads();
        float s[4][2] = {};
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
            float4 kv[2];
#pragma unroll
            for (int c = 0; c < 2; c++) kv[c] = *reinterpret_cast<const float4*>(ks + (tx + 16 * c) * QP + d);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float4 qv = *reinterpret_cast<const float4*>(qs + (4 * ty + r) * QP + d);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    s[r][c] = fmaf(qv.x, kv[c].x, s[r][c]);
                    s[r][c] = fmaf(qv.y, kv[c].y, s[r][c]);
                    s[r][c] = fmaf(qv.z, kv[c].z, s[r][c]);
                    s[r][c] = fmaf(qv.w, kv[c].w, s[r][c]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int c = 0; c < 2; c++) sc[(4 * ty + r) * SP + tx + 16 * c] = s[r][c];
        __syncthreads();
        // online softmax: a warp per row, lane = column
        for (int r = wid; r < AS_TM; r += AS_THREADS / WARP) {
            const int j = j0 + lane;
            const int p = a.qsl ? t.ctx + (t.r0 + r) / a.G : t.p0;
            const bool see = r < t.nr && j <= p && (a.window == 0 || j > p - a.window || j < a.sinks);
            const float x = see ? sc[r * SP + lane] : -INFINITY;
            const float mo = mrow[r], mn = fmaxf(mo, warp_max(x));
            const float w = see ? exp2f(x - mn) : 0.0f;
            const float sum = warp_sum(w);
            sc[r * SP + lane] = w;
            if (lane == 0) {
                const float corr = mo == -INFINITY ? 0.0f : exp2f(mo - mn);  // (nothing summed yet: nothing to scale)
                crow[r] = corr;
                lrow[r] = lrow[r] * corr + sum;
                mrow[r] = mn;
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float corr = crow[4 * ty + r];
#pragma unroll
            for (int i = 0; i < DV; i++) {
                acc[r][i].x *= corr;
                acc[r][i].y *= corr;
                acc[r][i].z *= corr;
                acc[r][i].w *= corr;
            }
        }
#pragma unroll 4
        for (int c = 0; c < AS_TN; c++) {
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; r++) w[r] = sc[(4 * ty + r) * SP + c];
#pragma unroll
            for (int i = 0; i < DV; i++) {
                const float4 v = *reinterpret_cast<const float4*>(vs + c * D + 4 * tx + 64 * i);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    acc[r][i].x = fmaf(w[r], v.x, acc[r][i].x);
                    acc[r][i].y = fmaf(w[r], v.y, acc[r][i].y);
                    acc[r][i].z = fmaf(w[r], v.z, acc[r][i].z);
                    acc[r][i].w = fmaf(w[r], v.w, acc[r][i].w);
                }
            }
        }
    }
    __syncthreads();
    if (a.n_splits > 1) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int row = 4 * ty + r;
            if (row >= t.nr) continue;
            const int64_t pr = part_row(a, grow(row), h, z, (t.r0 + row) % a.G);
#pragma unroll
            for (int i = 0; i < DV; i++) {                                   // (part_o need not be 16-byte aligned)
                float* o = a.part_o + pr * D + 4 * tx + 64 * i;
                o[0] = acc[r][i].x;
                o[1] = acc[r][i].y;
                o[2] = acc[r][i].z;
                o[3] = acc[r][i].w;
            }
            if (tx == 0) {
                // log2 units -> natural, for the combine; NaN scores leave the maximum as it was, +inf keeps the merge from dropping
                // their part
                const float l = lrow[row];
                a.part_ml[2 * pr] = l == l ? mrow[row] * 0.69314718055994531f : INFINITY;
                a.part_ml[2 * pr + 1] = l;
            }
        }
        return;
    }
    float* os = qs;                                                          // [TM][QP] the normalised output
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const float l = lrow[4 * ty + r], inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int i = 0; i < DV; i++)
            *reinterpret_cast<float4*>(os + (4 * ty + r) * QP + 4 * tx + 64 * i) =
                make_float4(acc[r][i].x * inv, acc[r][i].y * inv, acc[r][i].z * inv, acc[r][i].w * inv);
    }
    __syncthreads();
    IN* out = static_cast<IN*>(a.out);
    for (int r = wid; r < t.nr; r += AS_THREADS / WARP) {
        float x[R];
#pragma unroll
        for (int i = 0; i < R; i++) x[i] = os[r * QP + lane + WARP * i];
        if (a.rot) fwht_warp<D>(x, lane);
        IN* o = out + (grow(r) * a.H * a.G + head(r)) * D;
#pragma unroll
        for (int i = 0; i < R; i++) o[lane + WARP * i] = from_f32<IN>(x[i]);
    }
}

int launch_attend_simt(int D, int bits, int P, int dtype, const AttendArgs& a, int64_t rows, cudaStream_t stream) {
    // chunk: at most one tile more than rows * G / TM per sequence; decode: whole tiles of G rows per sequence
    const int64_t tiles = a.qsl ? (rows * a.G + AS_TM - 1) / AS_TM + a.S : int64_t(a.S) * ((a.G + AS_TM - 1) / AS_TM);
    if (tiles > 0x7fffffff || a.H > 65535 || a.n_splits > 65535)
        return set_error(KUSH_ERR_ARG, "attention: %lld row tiles, %d kv heads, %d splits", (long long)tiles, a.H, a.n_splits);
    return dispatch_fmt(D, bits, P, dtype, [&](auto Dc, auto Bc, auto Pc, auto in) {
        auto kern = attend_simt_kernel<Dc.value, Bc.value, Pc.value, decltype(in)>;
        constexpr int smem = AsSmem<Dc.value>::BYTES;
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return set_error(KUSH_ERR_CUDA, "attention: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
        launch_pdl(kern, dim3(unsigned(tiles), a.H, a.n_splits), dim3(AS_THREADS), size_t(smem), stream, a);
        return check_launch("attention (cuda cores)");
    });
}

}  // namespace kush
