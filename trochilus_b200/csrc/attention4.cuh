// attention4.cuh: a KV cache held in 4 bits, for several sequences on device rows: quantised as it is written, read
// back, attended to in full, or attended to in the blocks that a cheap score selects.
//
// A row is one position's key or value of one KV head (HD = 64 or 128 values) in groups of 32 consecutive values. A
// group holds a scale d and a minimum m (both f16) and a code 0..15 a value; a value reads back as f32(m + d code):
//   m = f16(min),  d = f16(max(0, max - m) / 15),  code = clamp(rint((x - m) / d), 0, 15), 0 where d is 0.
// Every rounding is of the real quotient (trx_a4_quant decides a quotient next to a border in 64 bits), so the codes do
// not depend on how they are computed. A group that holds a NaN or an infinity, or whose m or d passes f16, keeps
// d = NaN, m = 0 and codes 0: it reads back as NaN, and m is always finite.
//
// 64 positions of a (layer, sequence, KV head) are one record of contiguous memory (10240 bytes for HD 128: 5 bits a
// value), one bulk copy of the attention kernel:
//   keys    codes  [pos][c][g] one 32-bit word: dims 32 g + 8 c + j (j = 0..7) at bits 4 j        64 x HD / 2 bytes
//           d      [pos / 2][g][pos % 2] f16, m [pos][g] f16
//   values  codes  [pos / 8][n][c][g][odd] 16 bits (pos % 8 = 2 c + odd): dims 32 g + 4 n + i (i = 0..3) at bits 4 i
//           d, m   [pos / 2][g][pos % 2] f16
// The words are what a lane of a tensor-core fragment takes (the attention kernel's comment): no two positions share
// a byte of codes, so a position is written without reading its neighbours.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include "bulk.cuh"
#include "common.cuh"

#define TRX_A4_BLOCK 64 // positions a record

template <int HD> struct TrxA4L { // byte offsets in a record
    static constexpr int NG = HD / 32;
    static constexpr int KD = TRX_A4_BLOCK * HD / 2, KM = KD + TRX_A4_BLOCK * NG * 2;
    static constexpr int V = KM + TRX_A4_BLOCK * NG * 2, VD = V + KD, VM = V + KM;
    static constexpr int REC = 2 * V;
};

struct TrxA4 { // one layer of a session
    uint8_t *cache;  // [seq][KV head][block] records
    int8_t *bounds;  // [seq][KV head][block][HD / 8]{lowest of 8 dims, highest of 8 dims}
    float *units;    // [seq][KV head][block]
    int32_t *err;
    int64_t n_ctx;
    int n_blocks, n_seq, n_head, n_kv;
};

struct TrxA4Batch {
    const int32_t *slot, *pos0, *start; // start NULL: one row an entry
    int n_entries, n_tok, max_rows;
};

// what the session's error word says (the first that a kernel met; the entry is left out)
enum : int { TRX_A4_BAD_ENTRY = 1, TRX_A4_SAME_SLOT = 2, TRX_A4_GAVE_UP = 3 };

// Entry i of the batch: its sequence, first row, rows and first position. False: nothing to do (a padding entry or no
// rows, or an entry that passes the cache, the rows or max_rows, which is reported).
__device__ __forceinline__ bool trx_a4_entry(const TrxA4 &a, const TrxA4Batch &b, int i, int &slot, int &row0,
                                             int &rows, int &pos0) {
    slot = b.slot[i];
    if (slot < 0) return false;
    row0 = b.start ? b.start[i] : i;
    const int64_t r1 = b.start ? b.start[i + 1] : i + 1;
    const int64_t n = r1 - row0;
    pos0 = b.pos0[i];
    if (slot >= a.n_seq || row0 < 0 || n < 0 || r1 > b.n_tok || n > b.max_rows || pos0 < 0 || pos0 + n > a.n_ctx) {
        atomicCAS(a.err, 0, TRX_A4_BAD_ENTRY);
        return false;
    }
    rows = (int)n;
    return n > 0;
}

// 8 consecutive values of a row, as floats, and back
__device__ __forceinline__ void trx_a4_load8(const float *p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void trx_a4_load8(const __half *p, float (&x)[8]) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void trx_a4_load8(const __nv_bfloat16 *p, float (&x)[8]) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void trx_a4_store8(float *p, const float (&x)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ uint32_t trx_a4_pack2(float lo, float hi, const __half *) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t trx_a4_pack2(float lo, float hi, const __nv_bfloat16 *) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T> __device__ __forceinline__ void trx_a4_store8(T *p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(trx_a4_pack2(x[0], x[1], p), trx_a4_pack2(x[2], x[3], p),
                                               trx_a4_pack2(x[4], x[5], p), trx_a4_pack2(x[6], x[7], p));
}

// The 8 codes (4 bits each, value j at bits 4 j), scale and minimum of 8 values of a group whose other 24 lie in the
// lanes next to this one (4 aligned lanes a group; the whole warp calls).
// The quotient is taken in 32 bits, which is within 3 x 2^-24 x 22 < 4e-6 of the real one (a quotient is at most 15
// plus m's and d's roundings, below 22 even where d is a subnormal); one within 1e-5 of a border is taken again in
// 64 bits.
__device__ __forceinline__ uint32_t trx_a4_quant(const float (&x)[8], uint16_t &d16, uint16_t &m16) {
    float lo = x[0], hi = x[0];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        lo = fminf(lo, x[j]);
        hi = fmaxf(hi, x[j]);
        bad |= !(fabsf(x[j]) <= 3.402823466e38f);
    }
#pragma unroll
    for (int s = 1; s <= 2; s <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, s));
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, s) != 0;
    }
    const __half mh = __float2half_rn(lo);
    const float m = __half2float(mh);
    const __half dh = __double2half(__ddiv_rn(fmax(__dsub_rn((double)hi, (double)m), 0.0), 15.0));
    const float d = __half2float(dh);
    bad |= !(fabsf(m) <= 65504.0f) || !(d <= 65504.0f);
    d16 = bad ? (uint16_t)0x7fff : __half_as_ushort(dh);
    m16 = bad ? (uint16_t)0 : __half_as_ushort(mh);
    if (bad || d == 0.0f) return 0;
    const float rd = __fdiv_rn(1.0f, d);
    uint32_t codes = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float u = __fmul_rn(__fsub_rn(x[j], m), rd);
        float q = rintf(u);
        if (fabsf(u - q) > 0.49999f) q = (float)rint(__ddiv_rn(__dsub_rn((double)x[j], (double)m), (double)d));
        codes |= (uint32_t)(int)fminf(fmaxf(q, 0.0f), 15.0f) << (4 * j);
    }
    return codes;
}

// where lane a (dims 8 a .. 8 a + 7) of a row at position p of a record finds its codes, scale and minimum
template <int HD> __device__ __forceinline__ int trx_a4_kcode(int p, int a) {
    return p * (HD / 2) + ((a & 3) * TrxA4L<HD>::NG + (a >> 2)) * 4;
}
template <int HD> __device__ __forceinline__ int trx_a4_vcode(int p, int a, int half) { // dims 8 a + 4 half ..
    constexpr int NG = TrxA4L<HD>::NG;
    return TrxA4L<HD>::V + (p >> 3) * (4 * HD) + ((2 * (a & 3) + half) * 4 + ((p & 7) >> 1)) * (NG * 4) +
           (a >> 2) * 4 + (p & 1) * 2;
}
template <int HD> __device__ __forceinline__ int trx_a4_pair(int p, int g) { // in a [pos / 2][g][pos % 2] plane
    return (p >> 1) * (TrxA4L<HD>::NG * 4) + g * 4 + (p & 1) * 2;
}
template <int HD> __device__ __forceinline__ int trx_a4_km(int p, int g) {
    return TrxA4L<HD>::KM + p * (TrxA4L<HD>::NG * 2) + g * 2;
}

// 8 values (dims 8 a ..) of a key / value row
template <int HD> __device__ __forceinline__ void trx_a4_key8(const uint8_t *rec, int p, int a, float (&x)[8]) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(rec + trx_a4_kcode<HD>(p, a));
    const float d = trx_half(*reinterpret_cast<const uint16_t *>(rec + TrxA4L<HD>::KD + trx_a4_pair<HD>(p, a >> 2)));
    const float m = trx_half(*reinterpret_cast<const uint16_t *>(rec + trx_a4_km<HD>(p, a >> 2)));
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = __fmaf_rn(d, (float)((w >> (4 * j)) & 15), m); // (d x code is exact)
}
template <int HD> __device__ __forceinline__ void trx_a4_value8(const uint8_t *rec, int p, int a, float (&x)[8]) {
    const uint32_t w0 = *reinterpret_cast<const uint16_t *>(rec + trx_a4_vcode<HD>(p, a, 0));
    const uint32_t w1 = *reinterpret_cast<const uint16_t *>(rec + trx_a4_vcode<HD>(p, a, 1));
    const int s = trx_a4_pair<HD>(p, a >> 2);
    const float d = trx_half(*reinterpret_cast<const uint16_t *>(rec + TrxA4L<HD>::VD + s));
    const float m = trx_half(*reinterpret_cast<const uint16_t *>(rec + TrxA4L<HD>::VM + s));
#pragma unroll
    for (int j = 0; j < 4; j++) {
        x[j] = __fmaf_rn(d, (float)((w0 >> (4 * j)) & 15), m);
        x[4 + j] = __fmaf_rn(d, (float)((w1 >> (4 * j)) & 15), m);
    }
}

// Writes an entry's rows of one block (blockIdx.x blocks after the entry's first) and KV head (blockIdx.y), HD / 8
// lanes a row; then the block's bounds over all its 64 rows, which those rows may have changed: the lowest and highest
// key value of each dim as 8-bit multiples (floor, ceil, at most 127) of the block's unit, the power of two that puts
// their largest magnitude in [64, 128). A block with a NaN among its keys has the unit infinity. The rows that were
// never written count too; such a block is no earlier one of any query, so that its bounds are not read.
template <int HD, typename T>
__global__ void __launch_bounds__(256) trx_a4_write(TrxA4 a, TrxA4Batch b, const T *__restrict__ k, int64_t k_stride,
                                                    const T *__restrict__ v, int64_t v_stride) {
    constexpr int L = HD / 8, ROWS = 256 / L; // lanes a row, rows in flight
    __shared__ float s_lo[ROWS][HD], s_hi[ROWS][HD];
    __shared__ float s_max[HD / 32 + 1];
    int slot, row0, rows, pos0;
    const int tid = threadIdx.x, kv = blockIdx.y, e = blockIdx.z;
    if (!trx_a4_entry(a, b, e, slot, row0, rows, pos0)) return;
    const int blk = pos0 / TRX_A4_BLOCK + blockIdx.x, first = blk * TRX_A4_BLOCK;
    if (first >= pos0 + rows) return;
    int same = 0;
    for (int j = tid; j < e; j += 256) same |= b.slot[j] == slot;
    if (__syncthreads_or(same)) {
        if (tid == 0) atomicCAS(a.err, 0, TRX_A4_SAME_SLOT);
        return;
    }
    const int64_t at = ((int64_t)slot * a.n_kv + kv) * a.n_blocks + blk;
    uint8_t *rec = a.cache + at * TrxA4L<HD>::REC;
    const int p0 = max(pos0, first) - first, p1 = min(pos0 + rows - first, TRX_A4_BLOCK);
    const int l = tid % L, g = l >> 2;
    for (int base = p0; base < p1; base += ROWS) {
        const int p = base + tid / L;
        const bool on = p < p1;
        const int64_t row = row0 + (first + (on ? p : p0) - pos0);
        float x[8];
        uint16_t d, m;
        trx_a4_load8(k + row * k_stride + kv * HD + 8 * l, x);
        uint32_t c = trx_a4_quant(x, d, m);
        if (on) {
            *reinterpret_cast<uint32_t *>(rec + trx_a4_kcode<HD>(p, l)) = c;
            if ((l & 3) == 0) {
                *reinterpret_cast<uint16_t *>(rec + TrxA4L<HD>::KD + trx_a4_pair<HD>(p, g)) = d;
                *reinterpret_cast<uint16_t *>(rec + trx_a4_km<HD>(p, g)) = m;
            }
        }
        trx_a4_load8(v + row * v_stride + kv * HD + 8 * l, x);
        c = trx_a4_quant(x, d, m);
        if (on) {
            *reinterpret_cast<uint16_t *>(rec + trx_a4_vcode<HD>(p, l, 0)) = (uint16_t)c;
            *reinterpret_cast<uint16_t *>(rec + trx_a4_vcode<HD>(p, l, 1)) = (uint16_t)(c >> 16);
            if ((l & 3) == 0) {
                *reinterpret_cast<uint16_t *>(rec + TrxA4L<HD>::VD + trx_a4_pair<HD>(p, g)) = d;
                *reinterpret_cast<uint16_t *>(rec + TrxA4L<HD>::VM + trx_a4_pair<HD>(p, g)) = m;
            }
        }
    }
    __syncthreads();
    float lo[8], hi[8], x[8];
    int bad = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) lo[j] = INFINITY, hi[j] = -INFINITY;
    for (int p = tid / L; p < TRX_A4_BLOCK; p += ROWS) {
        trx_a4_key8<HD>(rec, p, l, x);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            lo[j] = fminf(lo[j], x[j]);
            hi[j] = fmaxf(hi[j], x[j]);
            bad |= x[j] != x[j];
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) s_lo[tid / L][8 * l + j] = lo[j], s_hi[tid / L][8 * l + j] = hi[j];
    bad = __syncthreads_or(bad);
    float l1 = 0.0f, h1 = 0.0f;
    if (tid < HD) {
        l1 = s_lo[0][tid], h1 = s_hi[0][tid];
        for (int r = 1; r < ROWS; r++) l1 = fminf(l1, s_lo[r][tid]), h1 = fmaxf(h1, s_hi[r][tid]);
        float most = fmaxf(fabsf(l1), fabsf(h1));
        for (int s = 16; s; s >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
        if ((tid & 31) == 0) s_max[tid >> 5] = most;
    }
    __syncthreads();
    if (tid < HD) {
        float most = s_max[0];
        for (int i = 1; i < HD / 32; i++) most = fmaxf(most, s_max[i]);
        int ex = 0;
        if (most > 0.0f && !bad) frexpf(most, &ex);
        // (keys are multiples of 2^-24 up to 65504 x 16: the unit is a normal float)
        const float unit = __int_as_float((ex - 7 + 127) << 23), per = __int_as_float((7 - ex + 127) << 23);
        int8_t *o = a.bounds + at * (2 * HD) + (tid >> 3) * 16 + (tid & 7);
        o[0] = bad ? 0 : (int8_t)fmaxf(floorf(__fmul_rn(l1, per)), -127.0f);
        o[8] = bad ? 0 : (int8_t)fminf(ceilf(__fmul_rn(h1, per)), 127.0f);
        if (tid == 0) a.units[at] = bad ? INFINITY : unit;
    }
}

// The rows of an entry's block read back (the write's grid)
template <int HD, typename T>
__global__ void __launch_bounds__(256) trx_a4_read(TrxA4 a, TrxA4Batch b, T *__restrict__ k, int64_t k_stride,
                                                   T *__restrict__ v, int64_t v_stride) {
    constexpr int L = HD / 8, ROWS = 256 / L;
    int slot, row0, rows, pos0;
    const int tid = threadIdx.x, kv = blockIdx.y;
    if (!trx_a4_entry(a, b, blockIdx.z, slot, row0, rows, pos0)) return;
    const int blk = pos0 / TRX_A4_BLOCK + blockIdx.x, first = blk * TRX_A4_BLOCK;
    const uint8_t *rec = a.cache + (((int64_t)slot * a.n_kv + kv) * a.n_blocks + blk) * TrxA4L<HD>::REC;
    const int p0 = max(pos0, first) - first, p1 = min(pos0 + rows - first, TRX_A4_BLOCK), l = tid % L;
    for (int p = p0 + tid / L; p < p1; p += ROWS) {
        const int64_t row = row0 + (first + p - pos0);
        float x[8];
        trx_a4_key8<HD>(rec, p, l, x);
        trx_a4_store8(k + row * k_stride + kv * HD + 8 * l, x);
        trx_a4_value8<HD>(rec, p, l, x);
        trx_a4_store8(v + row * v_stride + kv * HD + 8 * l, x);
    }
}

// ---------------------------------------------------------------------------------------------
// Attention: the simple form. A CTA a (query row, KV head); a head of the group after another: 8 warps take a listed
// block each in turn, lane l the dims 8 (l % (HD / 8)) of every second (fourth) position, with a running maximum and
// sum; the warps' results are joined through shared memory.
// list: the blocks to attend to (select), or NULL: blocks 0 .. n_list - 1.
template <int HD, typename T>
__device__ void trx_a4_attend_row(const TrxA4 &a, const uint8_t *recs, const int *list, int n_list, int pos,
                                  const T *q, float scale, T *out) {
    constexpr int L = HD / 8, PER = 32 / L, W = 8;
    __shared__ float s_m[W], s_l[W], s_o[W][HD];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, l = lane % L;
    float qx[8], o[8], x[8], m = -INFINITY, sum = 0.0f;
    trx_a4_load8(q + 8 * l, qx);
#pragma unroll
    for (int j = 0; j < 8; j++) o[j] = 0.0f;
    for (int i = warp; i < n_list; i += W) {
        const int blk = list ? list[i] : i;
        const uint8_t *rec = recs + (int64_t)blk * TrxA4L<HD>::REC;
        for (int p0 = 0; p0 < TRX_A4_BLOCK && blk * TRX_A4_BLOCK + p0 <= pos; p0 += PER) {
            const int p = p0 + lane / L;
            trx_a4_key8<HD>(rec, p, l, x);
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) s = __fmaf_rn(qx[j], x[j], s);
            for (int w = 1; w < L; w <<= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
            s *= scale;
            if (blk * TRX_A4_BLOCK + p > pos) continue; // (only lanes leave: the shuffles above are done)
            const float mn = fmaxf(m, s);
            // a NaN score makes the row NaN; -inf beside -inf adds nothing
            const float f = m == mn ? 1.0f : expf(m - mn), w = s == -INFINITY ? 0.0f : expf(s - mn);
            trx_a4_value8<HD>(rec, p, l, x);
            m = s != s ? s : mn;
            sum = __fmaf_rn(sum, f, w);
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = __fmaf_rn(w, x[j], o[j] * f);
        }
        __syncwarp();
    }
    (void)a;
    for (int w = L; w < 32; w <<= 1) { // the positions that lanes took side by side
        const float m2 = __shfl_xor_sync(0xffffffffu, m, w), sum2 = __shfl_xor_sync(0xffffffffu, sum, w);
        const float mn = fmaxf(m, m2), f = m == mn ? 1.0f : expf(m - mn), f2 = m2 == mn ? 1.0f : expf(m2 - mn);
        sum = sum * f + sum2 * f2;
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = o[j] * f + __shfl_xor_sync(0xffffffffu, o[j], w) * f2;
        m = mn;
    }
    __syncthreads(); // (the head before has been read)
    if (lane < L) {
        if (lane == 0) s_m[warp] = m, s_l[warp] = sum;
        for (int j = 0; j < 8; j++) s_o[warp][8 * l + j] = o[j];
    }
    __syncthreads();
    if (tid < L) {
        float M = -INFINITY, S = 0.0f;
        for (int w = 0; w < W; w++) M = fmaxf(M, s_m[w]);
        for (int j = 0; j < 8; j++) o[j] = 0.0f;
        for (int w = 0; w < W; w++) {
            const float f = s_m[w] == M ? 1.0f : expf(s_m[w] - M);
            S += s_l[w] * f;
            for (int j = 0; j < 8; j++) o[j] += s_o[w][8 * tid + j] * f;
        }
        for (int j = 0; j < 8; j++) o[j] = S == 0.0f ? 0.0f : __fdiv_rn(o[j], S);
        trx_a4_store8(out + 8 * tid, o);
    }
}

template <int HD, typename T>
__global__ void __launch_bounds__(256) trx_a4_attend(TrxA4 a, TrxA4Batch b, const T *__restrict__ q, int64_t q_stride,
                                                     float scale, T *__restrict__ out, int64_t out_stride) {
    int slot, row0, rows, pos0;
    const int kv = blockIdx.y, r = blockIdx.x, G = a.n_head / a.n_kv;
    if (!trx_a4_entry(a, b, blockIdx.z, slot, row0, rows, pos0) || r >= rows) return;
    const uint8_t *recs = a.cache + ((int64_t)slot * a.n_kv + kv) * a.n_blocks * TrxA4L<HD>::REC;
    const int pos = pos0 + r;
    for (int h = 0; h < G; h++)
        trx_a4_attend_row<HD, T>(a, recs, nullptr, pos / TRX_A4_BLOCK + 1, pos,
                                 q + (int64_t)(row0 + r) * q_stride + (kv * G + h) * HD, scale,
                                 out + (int64_t)(row0 + r) * out_stride + (kv * G + h) * HD);
}

// a float as an unsigned key of the same order (no NaN)
__device__ __forceinline__ uint32_t trx_a4_key(float f) {
    const uint32_t u = __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Attention to n_sel blocks: the row's own and the n_sel - 1 earlier ones of the best scores (ties to the lowest
// index). A block's score is f32(sum_i P_i highest_i + N_i lowest_i) x unit, an upper bound of the group's summed q.k
// in whole numbers: P_i and N_i sum the positive and the negative parts of the group's query values, which are rounded
// to multiples of a power of two that puts the largest magnitude in [64, 128) and kept within 127. Sums of whole
// numbers do not depend on their order, so neither does the selection. A block with a NaN among its keys scores +inf;
// a query with one selects by index. blocks (optional): the selected blocks, ascending, then -1.
template <int HD, typename T>
__global__ void __launch_bounds__(256) trx_a4_select(TrxA4 a, TrxA4Batch b, const T *__restrict__ q, int64_t q_stride,
                                                     float scale, int n_sel, T *__restrict__ out, int64_t out_stride,
                                                     int32_t *__restrict__ blocks) {
    constexpr int L = HD / 8;
    extern __shared__ uint32_t s_key[]; // [n_blocks] keys, then [n_sel] selected blocks
    __shared__ int s_p[HD], s_n[HD], s_cnt, s_wsum[8];
    __shared__ float s_max;
    int slot, row0, rows, pos0;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kv = blockIdx.y, r = blockIdx.x, G = a.n_head / a.n_kv;
    if (!trx_a4_entry(a, b, blockIdx.z, slot, row0, rows, pos0) || r >= rows) return;
    const int pos = pos0 + r, home = pos / TRX_A4_BLOCK;
    const int64_t at = ((int64_t)slot * a.n_kv + kv) * a.n_blocks;
    const T *qr = q + (int64_t)(row0 + r) * q_stride + kv * G * HD;
    int *list = reinterpret_cast<int *>(s_key + a.n_blocks);
    int n_list = home + 1;
    if (n_list > n_sel) {
        float most = 0.0f;
        int bad = 0;
        for (int i = tid; i < G * HD; i += 256) {
            const float f = fabsf((float)qr[i]);
            bad |= !(f <= 3.402823466e38f);
            most = fmaxf(most, f);
        }
        bad = __syncthreads_or(bad);
        for (int s = 16; s; s >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
        if (lane == 0) s_wsum[warp] = __float_as_int(most);
        __syncthreads();
        if (tid == 0) {
            for (int i = 1; i < 8; i++) most = fmaxf(most, __int_as_float(s_wsum[i]));
            s_max = most;
        }
        __syncthreads();
        most = s_max;
        if (tid < HD) {
            int ex = 0, up = 0, down = 0;
            if (most > 0.0f && !bad) frexpf(most, &ex);
            for (int h = 0; h < G; h++) {
                const float f = (float)qr[h * HD + tid];
                const int z = bad ? 0 : (int)fminf(fmaxf(rintf(ldexpf(f, 7 - ex)), -127.0f), 127.0f);
                up += max(z, 0);
                down += min(z, 0);
            }
            s_p[tid] = up, s_n[tid] = down;
        }
        __syncthreads();
        const int l = tid % L;
        for (int i0 = 0; i0 < home; i0 += 256 / L) {
            const int i = i0 + tid / L;
            int sum = 0;
            if (i < home) {
                const int8_t *w = a.bounds + (at + i) * (2 * HD) + l * 16;
                for (int j = 0; j < 8; j++) sum += s_n[8 * l + j] * w[j] + s_p[8 * l + j] * w[8 + j];
            }
            for (int s = 1; s < L; s <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
            if (i < home && l == 0) {
                const float u = a.units[at + i];
                s_key[i] = trx_a4_key(u == INFINITY ? INFINITY : __fmul_rn((float)sum, u));
            }
        }
        __syncthreads();
        // the largest key that at least want blocks reach
        const int want = n_sel - 1;
        uint32_t t = 0;
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t c = t | (1u << bit);
            int n = 0;
            for (int i = tid; i < home; i += 256) n += s_key[i] >= c;
            if (tid == 0) s_cnt = 0;
            __syncthreads();
            atomicAdd(&s_cnt, n);
            __syncthreads();
            if (s_cnt >= want) t = c;
            __syncthreads();
        }
        if (tid == 0) { // ascending: all above t, and the first ones at t
            int above = 0, n = 0;
            for (int i = 0; i < home; i++) above += s_key[i] > t;
            int ties = want - above;
            for (int i = 0; i < home; i++)
                if (s_key[i] > t || (s_key[i] == t && ties-- > 0)) list[n++] = i;
            list[n] = home;
        }
        n_list = n_sel;
    } else {
        for (int i = tid; i < n_list; i += 256) list[i] = i;
    }
    __syncthreads();
    if (blocks)
        for (int i = tid; i < n_sel; i += 256)
            blocks[((int64_t)(row0 + r) * a.n_kv + kv) * n_sel + i] = i < n_list ? list[i] : -1;
    const uint8_t *recs = a.cache + at * TrxA4L<HD>::REC;
    for (int h = 0; h < G; h++)
        trx_a4_attend_row<HD, T>(a, recs, list, n_list, pos, qr + h * HD, scale,
                                 out + (int64_t)(row0 + r) * out_stride + (kv * G + h) * HD);
}
