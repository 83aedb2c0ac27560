// Rotary positions of q and k rows: pair i of a head's first rotary_dim channels turns by positions[row] * f_i,
//   y1 = factor (x1 cos a - x2 sin a),  y2 = factor (x2 cos a + x1 sin a),
// pairs (i, i + rotary_dim / 2) or, interleaved, (2i, 2i + 1); the other channels pass through.
//
// Angles.  No cosine table is read: a frequency comes as turns per position in 64-bit fixed point, T_i = f_i / (2 pi)
// * 2^64, so position * T_i modulo 2^64 (one wrapping integer multiply) is the angle's fraction of a turn, exact range
// reduction included for every position; read as a signed number it lies in [-1/2, 1/2) turn and goes to sincospif
// after one rounding to fp32.  A far position loses nothing (|error| <= |position| 2^-65 turns: T_i is the nearest integer).
//
// Bound: HBM (each row read once, written once).  A block computes the cosines and sines of its rows once, into
// shared memory, and every thread keeps those of its pairs in registers while it walks the heads, two 16-byte vectors
// (a pair of half-vectors, or two interleaved ones) per head; rotary dims or addresses that 16-byte vectors do not
// divide take the same code one element at a time.  16384 rows of 32 + 8 heads of 128, bf16: 65.4 us, 5.1 TB/s = 78% of the
// measured copy rate; one row 2 us on the device, below the host's cost of a call (10 us).
#include "kush_common.cuh"

namespace kush {

constexpr int ROPE_THREADS = 256;

struct RopeRows {
    const void* x;
    void* y;
    int64_t xr, xh, yr, yh;        // row and head strides, in elements
    int heads;
};

template <class IN, int VE>
struct alignas(sizeof(IN) * VE) Vec {
    IN e[VE];
};

// a vector read once and written once: streaming loads and stores (16384 rows of 40 heads: 68.0 us without, 65.3 with)
template <class V> __device__ __forceinline__ V load_once(const V* p) {
    if constexpr (sizeof(V) == 16) {
        V v;
        *reinterpret_cast<uint4*>(&v) = __ldcs(reinterpret_cast<const uint4*>(p));
        return v;
    } else {
        return *p;
    }
}
template <class V> __device__ __forceinline__ void store_once(V* p, const V& v) {
    if constexpr (sizeof(V) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
    else *p = v;
}

// grid (ceil(rows / rpb)), block 256 = [rpb rows][head lanes][D / (2 VE) items]; an item is a pair of VE-element vectors
// of one head.  rpb: rows of a block, a power of two.
template <class IN, int VE, bool INTER>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(RopeRows qr, RopeRows kr, const void* __restrict__ positions,
                                                            int pos64, const uint64_t* __restrict__ turns, int D, int r,
                                                            float factor, int64_t rows, int rpb) {
    extern __shared__ float2 cs[];                              // [rpb][r / 2] factor * (cos, sin)
    pdl_wait();
    pdl_trigger();
    const int half = r / 2;
    const int64_t row0 = int64_t(blockIdx.x) * rpb;
    for (int i = threadIdx.x; i < rpb * half; i += ROPE_THREADS) {
        const int64_t row = row0 + i / half;
        if (row < rows) {
            const int64_t p = pos64 ? static_cast<const int64_t*>(positions)[row] : static_cast<const int32_t*>(positions)[row];
            const long long a = static_cast<long long>(uint64_t(p) * turns[i % half]);
            float sn, cn;
            sincospif(__ll2float_rn(a) * 0x1p-63f, &sn, &cn);    // 2^-64 turns -> half turns
            cs[i] = make_float2(factor * cn, factor * sn);
        }
    }
    __syncthreads();
    const int items = D / (2 * VE), nrot = r / (2 * VE);        // items below nrot are rotated, the others copied
    const int item = threadIdx.x % items, slot = threadIdx.x / items;
    const int rl = slot % rpb, hl = slot / rpb, nhl = ROPE_THREADS / items / rpb;
    const int64_t row = row0 + rl;
    if (row >= rows) return;
    // channels of the item's two vectors, and its pairs' first index
    const bool rot = item < nrot;
    const int c0 = !rot ? r + (item - nrot) * 2 * VE : INTER ? item * 2 * VE : item * VE;
    const int c1 = !rot || INTER ? c0 + VE : half + c0;
    float2 w[VE];
#pragma unroll
    for (int e = 0; e < VE; e++) w[e] = rot ? cs[rl * half + item * VE + e] : make_float2(1.0f, 0.0f);
    auto turn = [&](Vec<IN, VE>& a, Vec<IN, VE>& b) {
        if constexpr (INTER && VE > 1) {
#pragma unroll
            for (int e = 0; e < VE; e++) {                      // pair e: two neighbours of the 2 VE elements
                Vec<IN, VE>& v = e < VE / 2 ? a : b;
                const int i = 2 * (e % (VE / 2));
                const float x1 = to_f32(v.e[i]), x2 = to_f32(v.e[i + 1]);
                v.e[i] = from_f32<IN>(x1 * w[e].x - x2 * w[e].y);
                v.e[i + 1] = from_f32<IN>(x2 * w[e].x + x1 * w[e].y);
            }
        } else {
#pragma unroll
            for (int e = 0; e < VE; e++) {
                const float x1 = to_f32(a.e[e]), x2 = to_f32(b.e[e]);
                a.e[e] = from_f32<IN>(x1 * w[e].x - x2 * w[e].y);
                b.e[e] = from_f32<IN>(x2 * w[e].x + x1 * w[e].y);
            }
        }
    };
    using V = Vec<IN, VE>;
    auto walk = [&](const RopeRows& t) {
        const IN* x = static_cast<const IN*>(t.x) + row * t.xr;
        IN* y = static_cast<IN*>(t.y) + row * t.yr;
        const bool skip = !rot && t.x == t.y && t.xr == t.yr && t.xh == t.yh;      // in place: the rest is there
        if (skip) return;
#pragma unroll 4
        for (int h = hl; h < t.heads; h += nhl) {
            const IN* xs = x + h * t.xh;
            IN* ys = y + h * t.yh;
            V a = load_once(reinterpret_cast<const V*>(xs + c0)), b = load_once(reinterpret_cast<const V*>(xs + c1));
            if (rot) turn(a, b);
            store_once(reinterpret_cast<V*>(ys + c0), a);
            store_once(reinterpret_cast<V*>(ys + c1), b);
        }
    };
    walk(qr);
    walk(kr);
}

template <class IN, int VE>
static int launch_rope(const RopeRows& q, const RopeRows& k, const void* positions, int pos64, const uint64_t* turns, int D,
                       int r, bool inter, float factor, int64_t rows, cudaStream_t stream) {
    // eight rows a block once that fills every SM: angles of eight rows for one barrier, more heads per thread (16384 rows of
    // 40 heads, bf16: 1 row a block 98 us, 2 81, 4 65.3, 8 64.5, 16 68; 51.3 at the measured copy rate); one row a block below
    const int slots = ROPE_THREADS / (D / (2 * VE));
    int rpb = rows >= 8 * 148 ? 8 : 1;
    while (rpb > slots) rpb /= 2;
    const int64_t blocks = (rows + rpb - 1) / rpb;
    if (blocks > 0x7fffffff) return set_error(KUSH_ERR_ARG, "kush_sm100_rope: %lld rows", (long long)rows);
    const size_t smem = sizeof(float2) * size_t(rpb) * (r / 2);
    if (inter)
        launch_pdl(rope_kernel<IN, VE, true>, dim3(unsigned(blocks)), dim3(ROPE_THREADS), smem, stream, q, k, positions,
                   pos64, turns, D, r, factor, rows, rpb);
    else
        launch_pdl(rope_kernel<IN, VE, false>, dim3(unsigned(blocks)), dim3(ROPE_THREADS), smem, stream, q, k, positions,
                   pos64, turns, D, r, factor, rows, rpb);
    return check_launch("kush_sm100_rope");
}

}  // namespace kush

using namespace kush;

extern "C" int kush_sm100_rope(int32_t head_dim, int32_t dtype, int32_t rotary_dim, int32_t interleaved, const void* q,
                               int64_t q_row_stride, int64_t q_head_stride, void* q_out, int64_t qo_row_stride,
                               int64_t qo_head_stride, int32_t q_heads, const void* k, int64_t k_row_stride,
                               int64_t k_head_stride, void* k_out, int64_t ko_row_stride, int64_t ko_head_stride,
                               int32_t k_heads, const void* positions, int32_t positions_64, const uint64_t* turns,
                               float factor, int64_t rows, void* stream) {
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return set_error(KUSH_ERR_UNSUPPORTED, "kush_sm100_rope: head_dim %d", head_dim);
    if (rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2)
        return set_error(KUSH_ERR_ARG, "kush_sm100_rope: rotary_dim %d must be even and in [2, %d]", rotary_dim, head_dim);
    if (rows < 0 || q_heads < 0 || k_heads < 0)
        return set_error(KUSH_ERR_ARG, "kush_sm100_rope: rows %lld q_heads %d k_heads %d", (long long)rows, q_heads, k_heads);
    if (rows == 0 || q_heads + int64_t(k_heads) == 0) return KUSH_OK;
    if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || !positions || !turns)
        return set_error(KUSH_ERR_ARG, "kush_sm100_rope: null pointer");
    const RopeRows qr{q, q_out, q_row_stride, q_head_stride, qo_row_stride, qo_head_stride, q_heads};
    const RopeRows kr{k, k_out, k_row_stride, k_head_stride, ko_row_stride, ko_head_stride, k_heads};
    const int rc = dispatch_dtype(dtype, [&](auto in) {
        using IN = decltype(in);
        constexpr int VE = 16 / sizeof(IN);
        auto vec = [](const RopeRows& t) {                      // every vector of the rows is 16-byte aligned
            return t.heads == 0 || (aligned16(t.x) && aligned16(t.y) && ((t.xr | t.xh | t.yr | t.yh) % VE) == 0);
        };
        const bool wide = rotary_dim % (2 * VE) == 0 && vec(qr) && vec(kr);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        return wide ? launch_rope<IN, VE>(qr, kr, positions, positions_64, turns, head_dim, rotary_dim, interleaved != 0,
                                          factor, rows, st)
                    : launch_rope<IN, 1>(qr, kr, positions, positions_64, turns, head_dim, rotary_dim, interleaved != 0,
                                         factor, rows, st);
    });
    if (rc == KUSH_ERR_UNSUPPORTED) return set_error(rc, "kush_sm100_rope: dtype %d", dtype);
    return rc;
}
