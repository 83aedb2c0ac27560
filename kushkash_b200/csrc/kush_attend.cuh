// What the kernels of chunk attention (several query rows per sequence over the cached history and the new rows) share:
// the arguments, the mapping of a block to a tile of query rows, and the tiles of keys that tile sees.
//
// Query rows of (sequence s, kv head h) are flattened as r = t * G + g: new token t (position ctx + t), q head h * G + g.
// A tile is TM consecutive rows of one sequence.  Positions [0, ctx) are cached (full pages in records, the unfinished
// page's keys in tail_k), positions [ctx, ctx + new) are the new rows.
#pragma once

#include "kush_common.cuh"

namespace kush {

constexpr int32_t KUSH_NO_POSITION = 1 << 30;      // above every position

struct AttendArgs {
    const void* q;
    void* out;
    const void* k_new;               // null: every key is in the cache, the queries are at its last position (decode)
    const void* v_new;
    int64_t q_stride, k_stride, v_stride;
    const uint8_t* cache;
    int64_t block_stride, head_stride;
    const void* tail_k;
    const int32_t *tail_idx, *block_table, *seq_lens, *qsl;      // qsl null in decode
    int64_t max_pages;
    int32_t H, G, S;
    int32_t n_rows;                  // rows of q, k_new and v_new (query_start_loc is not believed beyond them)
    float sm_log2;                   // scale * log2(e)
    int32_t window, sinks;           // window 0: none
    int32_t n_splits;
    float *part_ml, *part_o;
    int32_t rot;                     // decode with rotation: q rotated as it loads, the output rotated back
    // limit_ms > 0: this slot of every block keeps back its tile-th tile's weights, and waits end after limit_ms
    struct { int32_t slot, tile, limit_ms; } held;
};

struct RowTile {
    int s;               // sequence
    int r0, nr;          // its flattened rows [r0, r0 + nr)
    int64_t q0;          // global row of its token 0
    int ctx, n_new;      // cached tokens, new tokens
    int p0, p1;          // positions of the tile's first and last row
};

// tile x of the launch, false if there is none; every warp computes it (sequences 32 at a time)
__device__ __forceinline__ bool row_tile(const AttendArgs& a, int x, int TM, RowTile& t) {
    if (a.qsl == nullptr) {                                       // decode: G rows per sequence at its last token
        const int per = (a.G + TM - 1) / TM;
        t.s = x / per;
        if (t.s >= a.S) return false;
        t.r0 = (x % per) * TM;
        t.nr = min(TM, a.G - t.r0);
        t.q0 = t.s;
        t.ctx = a.seq_lens[t.s];
        t.n_new = 0;
        t.p0 = t.p1 = t.ctx - 1;
        return true;
    }
    const int lane = threadIdx.x % WARP;
    int base = 0;
    for (int i0 = 0; i0 < a.S; i0 += WARP) {
        const int i = i0 + lane;
        const int n = i < a.S ? max(0, min(a.qsl[i + 1], a.n_rows) - max(0, a.qsl[i])) : 0;
        const int cnt = int((int64_t(n) * a.G + TM - 1) / TM);
        int sum = cnt;
#pragma unroll
        for (int o = 1; o < WARP; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + sum > x);
        if (past) {
            const int l = __ffs(past) - 1;
            t.s = i0 + l;
            t.n_new = __shfl_sync(0xffffffffu, n, l);
            t.r0 = (x - base - __shfl_sync(0xffffffffu, sum - cnt, l)) * TM;
            t.nr = int(min(int64_t(TM), int64_t(t.n_new) * a.G - t.r0));
            t.q0 = max(0, a.qsl[t.s]);
            t.ctx = max(0, a.seq_lens[t.s] - t.n_new);
            t.p0 = t.ctx + t.r0 / a.G;
            t.p1 = t.ctx + (t.r0 + t.nr - 1) / a.G;
            return true;
        }
        base += __shfl_sync(0xffffffffu, sum, WARP - 1);
    }
    return false;
}

// The key tiles (TN tokens, aligned) that some row of a tile of rows sees: tiles [0, a) hold the sinks, [b, e) the
// window.  Token j is seen by some row iff j <= p1 and (j >= lo or j < ns).
struct KeyTiles {
    int lo, ns;
    int a, b, count;
    __device__ __forceinline__ int tile(int i) const { return i < a ? i : i - a + b; }
    __device__ __forceinline__ bool seen(int j, int p1) const { return j <= p1 && (j >= lo || j < ns); }
};

__device__ __forceinline__ KeyTiles key_tiles(int p0, int p1, int window, int sinks, int TN) {
    KeyTiles k;
    k.lo = window > 0 ? max(0, p0 - window + 1) : 0;
    k.ns = min(sinks, k.lo);
    k.b = k.lo / TN;
    k.a = min((k.ns + TN - 1) / TN, k.b);
    k.count = p1 < 0 ? 0 : k.a + p1 / TN + 1 - k.b;
    return k;
}

// Split z of a row tile owns its key tiles [i0, i1): one quota for the batch, from an upper bound of the count over the
// sequences, so that the splits go to the long sequences of a ragged batch.  Every warp computes it.
__device__ __forceinline__ void key_split(const AttendArgs& a, int z, int TM, int TN, int count, int& i0, int& i1) {
    if (a.n_splits == 1) {
        i0 = 0;
        i1 = count;
        return;
    }
    int mx = 0;
    for (int i = threadIdx.x % WARP; i < a.S; i += WARP) mx = max(mx, a.seq_lens[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    int64_t bound = (int64_t(mx) + TN - 1) / TN;
    if (a.window > 0) {
        const int64_t span = TM / a.G + 2;                        // tokens a tile of rows can reach over
        bound = min(bound, (a.window + span) / TN + 2 + (int64_t(a.sinks) + TN - 1) / TN);
    }
    const int quota = max(1, int((bound + a.n_splits - 1) / a.n_splits));
    i0 = int(min(int64_t(count), int64_t(z) * quota));
    i1 = min(count, i0 + quota);
}

// partial row index of (global row, kv head, split, g): the layout of kush_sm100_combine with a row for a sequence
__device__ __forceinline__ int64_t part_row(const AttendArgs& a, int64_t row, int h, int z, int g) {
    return ((row * a.H + h) * a.n_splits + z) * a.G + g;
}

// the tensor-core kernel (kush_attend_tc.cu): fp16 / bf16 rows, head_dim 64 or 128, any group
int attend_tc_supported(int D, int dtype);
int launch_attend_tc(int D, int bits, int P, int dtype, const AttendArgs& a, int64_t rows, cudaStream_t stream);
int launch_attend_simt(int D, int bits, int P, int dtype, const AttendArgs& a, int64_t rows, cudaStream_t stream);
// the merge of split partials into a.out (out, part_ml, part_o, n_splits, H, G, qsl, S of a); part_ml 8-byte, part_o 16-byte aligned
int launch_chunk_combine(int D, int dtype, const AttendArgs& a, int64_t rows, cudaStream_t stream);

}  // namespace kush
