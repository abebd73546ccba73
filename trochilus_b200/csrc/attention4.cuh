// attention4.cuh: a KV cache held in 4 bits, for several sequences on device rows: quantised as it is written, read
// back, attended to in full, or attended to in the blocks that a cheap score selects.
//
// A row is one position's key or value of one KV head (HD = 64 or 128 values) in groups of 32 consecutive values. A
// group holds a scale d and a minimum m (both f16) and a code 0..15 a value; a value reads back as f32(m + d code):
//   m = f16(min),  d = f16(max(0, max - m) / 15),  code = clamp(rint((x - m) / d), 0, 15), 0 where d is 0.
// Every rounding is of the real quotient (trx_a4_quant decides a quotient next to a border exactly), so the codes do
// not depend on how they are computed. A group that holds a NaN or an infinity, or whose m or d passes f16, keeps
// d = NaN, m = 0 and codes 0: it reads back as NaN, and m is always finite.
//
// 32 positions of a (layer, sequence, KV head) are one record of contiguous memory (5120 bytes for HD 128: 5 bits a
// value):
//   keys    codes  [pos][c][g] one 32-bit word: dims 32 g + 8 c + j (j = 0..7) at bits 4 j        32 x HD / 2 bytes
//           d, m   [pos][g] f16
//   values  codes  [pos / 8][n][c][g][odd] 16 bits (pos % 8 = 2 c + odd): dims 32 g + 4 n + i (i = 0..3) at bits 4 i
//           d, m   [pos / 2][g][pos % 2] f16
// The words are what a lane of a tensor-core fragment takes (the attention kernel's comment): no two positions share
// a byte of codes, so a position is written without reading its neighbours. Two records are a block of 64 positions,
// the unit of selection.
#pragma once
#include <climits>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include "bulk.cuh"
#include "common.cuh"

#define TRX_A4_REC 32   // positions a record
#define TRX_A4_BLOCK 64 // positions a block

template <int HD> struct TrxA4L { // byte offsets in a record
    static constexpr int NG = HD / 32;
    static constexpr int KD = TRX_A4_REC * HD / 2, KM = KD + TRX_A4_REC * NG * 2;
    static constexpr int V = KM + TRX_A4_REC * NG * 2, VD = V + KD, VM = V + KM;
    static constexpr int REC = 2 * V, BLOCK = 2 * REC;
};

struct TrxA4 { // one layer of a session
    uint8_t *cache;  // [seq][KV head][block] two records each
    int8_t *bounds;  // [seq][KV head][block][2][HD]: lowest, then highest
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
    pos0 = b.pos0[i];
    row0 = b.start ? b.start[i] : i;
    const int64_t r1 = b.start ? b.start[i + 1] : i + 1;
    const int64_t n = r1 - row0;
    if (slot < 0) return false;
    if (slot >= a.n_seq || row0 < 0 || n < 0 || r1 > b.n_tok || n > b.max_rows || pos0 < 0 || pos0 + n > a.n_ctx) {
        atomicCAS(a.err, 0, TRX_A4_BAD_ENTRY);
        return false;
    }
    rows = (int)n;
    return n > 0;
}

// 8 consecutive values of a row: as they lie in memory, as floats, and back
template <typename T> struct TrxA4Raw {
    uint4 w[sizeof(T) / 2];
};
template <typename T> __device__ __forceinline__ TrxA4Raw<T> trx_a4_raw8(const T *p) {
    TrxA4Raw<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) r.w[i] = reinterpret_cast<const uint4 *>(p)[i];
    return r;
}
__device__ __forceinline__ void trx_a4_floats(const TrxA4Raw<float> &r, float (&x)[8]) {
    const uint32_t u[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __uint_as_float(u[i]);
}
__device__ __forceinline__ void trx_a4_floats(const TrxA4Raw<__half> &r, float (&x)[8]) {
    const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void trx_a4_floats(const TrxA4Raw<__nv_bfloat16> &r, float (&x)[8]) {
    const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
template <typename T> __device__ __forceinline__ void trx_a4_load8(const T *p, float (&x)[8]) {
    trx_a4_floats(trx_a4_raw8(p), x);
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

// three-operand minimum and maximum (a NaN beside a number is dropped; _nan: stays)
__device__ __forceinline__ float trx_a4_min3(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float trx_a4_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float trx_a4_max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// codes with those whose quotient is within `near` of a border (or of what 32 bits tell apart from one) taken exactly
// (seldom called, and kept out of the loops): x is compared with the border m + (k + 1/2) d itself, whose second term is
// exact: with its nearest float s, and where x is s, with what s dropped. (The last border is 14.5 d: a scale rounded down
// among f16's smallest numbers leaves quotients up to 22, and codes stay 15.)
__device__ __noinline__ uint32_t trx_a4_near(float x0, float x1, float x2, float x3, float x4, float x5, float x6, float x7, float m,
                                             float d, float rd, float near, uint32_t codes) {
    const float x[8] = {x0, x1, x2, x3, x4, x5, x6, x7};
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float u = __saturatef(__fmul_rn(__fsub_rn(x[j], m), rd)) * 15.0f;
        const float k = fminf(floorf(u), 14.0f);
        if (fabsf(__fsub_rn(__fsub_rn(u, k), 0.5f)) > 2.0f * near) continue;
        const float h = __fmul_rn(__fadd_rn(k, 0.5f), d), s = __fadd_rn(m, h);
        const float t = __fsub_rn(s, m); // s + lost = m + h
        const float lost = __fadd_rn(__fsub_rn(m, __fsub_rn(s, t)), __fsub_rn(h, t));
        const bool up = x[j] > s || (x[j] == s && (lost < 0.0f || (lost == 0.0f && ((int)k & 1))));
        codes = (codes & ~(15u << (4 * j))) | (uint32_t)((int)k + up) << (4 * j);
    }
    return codes;
}

// The 8 codes (4 bits each, value j at bits 4 j), scale and minimum of 8 values of a group whose other 24 lie in the
// lanes next to this one (4 aligned lanes a group; the whole warp calls). VALUES: x becomes what they stand for.
// Both are taken in 32 bits, and exactly where that may round to another side. (hi - m) / 15 is off by less than 2^-22 of
// itself, so it is certain unless 1 - 2^-21 and 1 + 2^-21 times it round apart (then: in 64 bits). A quotient, kept within
// 0 .. 15, is 15 times the saturated x r - m r, r = 1 / (15 d) (15 d is exact): off by less than 4 x 2^-24 x 15 < 4e-6
// where m r is small, and by the rounding of m r, 15 x 2^-24 |m r|, where it is not: it is certain unless it is within
// near = 1e-5 + 2^-19 |m r| of a border. (16-bit inputs meet borders often.)
template <bool VALUES> __device__ __forceinline__ uint32_t trx_a4_quant(float (&x)[8], uint16_t &d16, uint16_t &m16) {
    float lo = trx_a4_min3(x[0], x[1], x[2]), hi = trx_a4_max3_nan(x[0], x[1], x[2]);
    lo = trx_a4_min3(lo, x[3], x[4]), hi = trx_a4_max3_nan(hi, x[3], x[4]);
    lo = trx_a4_min3(lo, x[5], x[6]), hi = trx_a4_max3_nan(hi, x[5], x[6]);
    lo = fminf(lo, x[7]), hi = trx_a4_max3_nan(hi, hi, x[7]);
#pragma unroll
    for (int s = 1; s <= 2; s <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, s));
        hi = trx_a4_max3_nan(hi, hi, __shfl_xor_sync(0xffffffffu, hi, s));
    }
    const __half mh = __float2half_rn(lo);
    const float m = __half2float(mh);
    const float step = __fmul_rn(fmaxf(__fsub_rn(hi, m), 0.0f), 0.0666666701f);
    __half dh = __float2half_rn(__fmul_rn(step, 1.0f - 4.76837158e-7f));
    if (__half_as_ushort(dh) != __half_as_ushort(__float2half_rn(__fmul_rn(step, 1.0f + 4.76837158e-7f))))
        dh = __double2half(__ddiv_rn(fmax(__dsub_rn((double)hi, (double)m), 0.0), 15.0));
    const float d = __half2float(dh);
    // (an infinity among the values makes m or d one; a NaN leaves hi one)
    const bool bad = hi != hi || !(fabsf(m) <= 65504.0f) || !(d <= 65504.0f);
    d16 = bad ? (uint16_t)0x7fff : __half_as_ushort(dh);
    m16 = bad ? (uint16_t)0 : __half_as_ushort(mh);
    if (bad || d == 0.0f) {
        if constexpr (VALUES)
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = bad ? __int_as_float(0x7fffffff) : m;
        return 0;
    }
    const float r = __frcp_rn(__fmul_rn(15.0f, d)), mr = __fmul_rn(m, -r), near = __fmaf_rn(fabsf(mr), 1.9073486e-6f, 1.0e-5f);
    float q[8], far[8];
#pragma unroll
    for (int j = 0; j < 8; j++) { // (an integer's nearest: what 1.5 x 2^23 + 15 v keeps)
        const float v = __saturatef(__fmaf_rn(x[j], r, mr));
        q[j] = __fsub_rn(__fmaf_rn(v, 15.0f, 12582912.0f), 12582912.0f);
        far[j] = fabsf(__fmaf_rn(v, 15.0f, -q[j]));
    }
    // four codes are a number below 2^16, whose bits 8388608 + it holds
    const float c0 = __fmaf_rn(q[3], 4096.0f, __fmaf_rn(q[2], 256.0f, __fmaf_rn(q[1], 16.0f, q[0])));
    const float c1 = __fmaf_rn(q[7], 4096.0f, __fmaf_rn(q[6], 256.0f, __fmaf_rn(q[5], 16.0f, q[4])));
    uint32_t codes = __byte_perm(__float_as_uint(__fadd_rn(c0, 8388608.0f)), __float_as_uint(__fadd_rn(c1, 8388608.0f)), 0x5410);
    if (fmaxf(trx_a4_max3(trx_a4_max3(far[0], far[1], far[2]), far[3], far[4]), trx_a4_max3(far[5], far[6], far[7])) > 0.5f - near) {
        codes = trx_a4_near(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], m, d, r, near, codes);
        if constexpr (VALUES)
#pragma unroll
            for (int j = 0; j < 8; j++) q[j] = (float)((codes >> (4 * j)) & 15);
    }
    if constexpr (VALUES)
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __fmaf_rn(d, q[j], m); // (d x code is exact)
    return codes;
}

// where lane a (dims 8 a .. 8 a + 7) of a row at position p of a record finds its codes, scale and minimum (p up to 63:
// the block's second record)
template <int HD> __device__ __forceinline__ int trx_a4_kcode(int p, int a) {
    return (p >> 5) * TrxA4L<HD>::REC + (p & 31) * (HD / 2) + ((a & 3) * TrxA4L<HD>::NG + (a >> 2)) * 4;
}
template <int HD> __device__ __forceinline__ int trx_a4_vcode(int p, int a, int half) { // dims 8 a + 4 half ..
    constexpr int NG = TrxA4L<HD>::NG;
    return (p >> 5) * TrxA4L<HD>::REC + TrxA4L<HD>::V + ((p & 31) >> 3) * (4 * HD) +
           ((2 * (a & 3) + half) * 4 + ((p & 7) >> 1)) * (NG * 4) + (a >> 2) * 4 + (p & 1) * 2;
}
template <int HD> __device__ __forceinline__ int trx_a4_pair(int p, int g) { // in a [pos / 2][g][pos % 2] plane
    return (p >> 5) * TrxA4L<HD>::REC + ((p & 31) >> 1) * (TrxA4L<HD>::NG * 4) + g * 4 + (p & 1) * 2;
}
template <int HD> __device__ __forceinline__ int trx_a4_flat(int p, int g) { // in a [pos][g] plane
    return (p >> 5) * TrxA4L<HD>::REC + (p & 31) * (TrxA4L<HD>::NG * 2) + g * 2;
}

// 4 values of a group from 16 bits of codes, and 8 values (dims 8 a ..) of a key or value row
__device__ __forceinline__ void trx_a4_value4(uint32_t codes, float d, float m, float *x) {
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = __fmaf_rn(d, (float)((codes >> (4 * j)) & 15), m); // (d x code is exact)
}
template <int HD> __device__ __forceinline__ void trx_a4_key_scale(const uint8_t *rec, int p, int g, float &d, float &m) {
    d = trx_half(*reinterpret_cast<const uint16_t *>(rec + TrxA4L<HD>::KD + trx_a4_flat<HD>(p, g)));
    m = trx_half(*reinterpret_cast<const uint16_t *>(rec + TrxA4L<HD>::KM + trx_a4_flat<HD>(p, g)));
}
template <int HD> __device__ __forceinline__ void trx_a4_value_scale(const uint8_t *rec, int p, int g, float &d, float &m) {
    d = trx_half(*reinterpret_cast<const uint16_t *>(rec + TrxA4L<HD>::VD + trx_a4_pair<HD>(p, g)));
    m = trx_half(*reinterpret_cast<const uint16_t *>(rec + TrxA4L<HD>::VM + trx_a4_pair<HD>(p, g)));
}
template <int HD> __device__ __forceinline__ void trx_a4_key8(const uint8_t *rec, int p, int a, float (&x)[8]) {
    const uint32_t w = *reinterpret_cast<const uint32_t *>(rec + trx_a4_kcode<HD>(p, a));
    float d, m;
    trx_a4_key_scale<HD>(rec, p, a >> 2, d, m);
    trx_a4_value4(w & 0xffffu, d, m, x);
    trx_a4_value4(w >> 16, d, m, x + 4);
}
template <int HD> __device__ __forceinline__ void trx_a4_value8(const uint8_t *rec, int p, int a, float (&x)[8]) {
    float d, m;
    trx_a4_value_scale<HD>(rec, p, a >> 2, d, m);
    trx_a4_value4(*reinterpret_cast<const uint16_t *>(rec + trx_a4_vcode<HD>(p, a, 0)), d, m, x);
    trx_a4_value4(*reinterpret_cast<const uint16_t *>(rec + trx_a4_vcode<HD>(p, a, 1)), d, m, x + 4);
}

// Writes an entry's rows of one block (blockIdx.x blocks after the entry's first) and KV head (blockIdx.y), HD / 8
// lanes a row; and the block's bounds over all its 64 rows, which those rows may change: the lowest and highest key value
// of each dim as 8-bit multiples (floor, ceil, at most 127) of the block's unit, the power of two that puts their largest
// magnitude in [64, 128). A block with a NaN among its keys has the unit infinity. The rows that were never written
// count too; such a block is no earlier one of any query, so that its bounds are not read.
// The records are put together in shared memory (a row's value codes lie 2 bytes here and there) and leave it 16 bytes a
// thread where the block is written whole, else as the rows' own pieces.
// What bounds it: the quantiser's instructions. 4096 rows of 16 heads of 128 (f32, 77 MB): 22 us, 0.54 of the measured copy
// rate. Keys and values in CTAs of their own: 31 us against 29 then.
template <int HD, typename T>
__global__ void __launch_bounds__(256, 3) trx_a4_write(TrxA4 a, TrxA4Batch b, const T *__restrict__ k, int64_t k_stride,
                                                    const T *__restrict__ v, int64_t v_stride) {
    constexpr int L = HD / 8, ROWS = 256 / L, N = TRX_A4_BLOCK / ROWS; // lanes a row, rows in flight, passes
    using Y = TrxA4L<HD>;
    __shared__ __align__(16) uint8_t s_rec[Y::BLOCK];
    __shared__ float s_lo[8][HD], s_hi[8][HD];
    __shared__ float s_max[HD / 32];
    int slot, row0, rows, pos0;
    const int tid = threadIdx.x, kv = blockIdx.y, e = blockIdx.z;
    if (!trx_a4_entry(a, b, e, slot, row0, rows, pos0)) return;
    const int blk = pos0 / TRX_A4_BLOCK + blockIdx.x, first = blk * TRX_A4_BLOCK;
    if (first >= pos0 + rows) return;
    const int64_t at = ((int64_t)slot * a.n_kv + kv) * a.n_blocks + blk;
    uint8_t *rec = a.cache + at * Y::BLOCK;
    const int p0 = max(pos0, first) - first, p1 = min(pos0 + rows - first, TRX_A4_BLOCK);
    const int l = tid % L, g = l >> 2;
    for (int j = 0; j < e; j += 32) // (each warp looks for itself: no barrier before the rows)
        if (__any_sync(0xffffffffu, j + (tid & 31) < e && b.slot[j + (tid & 31)] == slot)) {
            if (tid == 0) atomicCAS(a.err, 0, TRX_A4_SAME_SLOT);
            return;
        }
    float lo[8], hi[8];
    int bad = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) lo[j] = INFINITY, hi[j] = -INFINITY;
#pragma unroll 1
    for (int i = 0; i < N; i += 2) { // two rows a lane
        int p[2];
        bool on[2];
        TrxA4Raw<T> rk[2], rv[2];
        float x[2][8];
        uint16_t d, m;
#pragma unroll
        for (int r = 0; r < 2; r++) {
            p[r] = (i + r) * ROWS + tid / L;
            on[r] = p[r] >= p0 && p[r] < p1;
            const int64_t row = row0 + (int64_t)(first + p[r] - pos0);
            if (on[r]) {
                rk[r] = trx_a4_raw8(k + row * k_stride + kv * HD + 8 * l);
                rv[r] = trx_a4_raw8(v + row * v_stride + kv * HD + 8 * l);
            } else rk[r] = rv[r] = TrxA4Raw<T>{};
        }
#pragma unroll
        for (int r = 0; r < 2; r++) {
            trx_a4_floats(rk[r], x[r]);
            if (__any_sync(0xffffffffu, on[r])) {
                const uint32_t c = trx_a4_quant<true>(x[r], d, m);
                if (on[r]) {
                    *reinterpret_cast<uint32_t *>(s_rec + trx_a4_kcode<HD>(p[r], l)) = c;
                    if ((l & 3) == 0) {
                        *reinterpret_cast<uint16_t *>(s_rec + Y::KD + trx_a4_flat<HD>(p[r], g)) = d;
                        *reinterpret_cast<uint16_t *>(s_rec + Y::KM + trx_a4_flat<HD>(p[r], g)) = m;
                    }
                }
            }
            if (!on[r]) trx_a4_key8<HD>(rec, p[r], l, x[r]); // a row that stays
            bad |= x[r][0] != x[r][0];                       // (a group's values are NaN together)
        }
#pragma unroll
        for (int j = 0; j < 8; j++) lo[j] = trx_a4_min3(lo[j], x[0][j], x[1][j]), hi[j] = trx_a4_max3(hi[j], x[0][j], x[1][j]);
#pragma unroll
        for (int r = 0; r < 2; r++)
            if (__any_sync(0xffffffffu, on[r])) {
                trx_a4_floats(rv[r], x[r]);
                const uint32_t c = trx_a4_quant<false>(x[r], d, m);
                if (on[r]) {
                    *reinterpret_cast<uint16_t *>(s_rec + trx_a4_vcode<HD>(p[r], l, 0)) = (uint16_t)c;
                    *reinterpret_cast<uint16_t *>(s_rec + trx_a4_vcode<HD>(p[r], l, 1)) = (uint16_t)(c >> 16);
                    if ((l & 3) == 0) {
                        *reinterpret_cast<uint16_t *>(s_rec + Y::VD + trx_a4_pair<HD>(p[r], g)) = d;
                        *reinterpret_cast<uint16_t *>(s_rec + Y::VM + trx_a4_pair<HD>(p[r], g)) = m;
                    }
                }
            }
    }
    // the lanes that share dims in a warp, then the warps
#pragma unroll
    for (int s = L; s < 32; s <<= 1)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            lo[j] = fminf(lo[j], __shfl_xor_sync(0xffffffffu, lo[j], s));
            hi[j] = fmaxf(hi[j], __shfl_xor_sync(0xffffffffu, hi[j], s));
        }
    if ((tid & 31) < L) {
#pragma unroll
        for (int j = 0; j < 8; j++) s_lo[tid >> 5][8 * l + j] = lo[j], s_hi[tid >> 5][8 * l + j] = hi[j];
    }
    bad = __syncthreads_or(bad);
    if (p0 == 0 && p1 == TRX_A4_BLOCK) {
        for (int i = tid; i < Y::BLOCK / 16; i += 256) reinterpret_cast<uint4 *>(rec)[i] = reinterpret_cast<const uint4 *>(s_rec)[i];
    } else {
        for (int p = p0 + tid / L; p < p1; p += ROWS) {
            auto copy = [&](int off, auto t) {
                using U = decltype(t);
                *reinterpret_cast<U *>(rec + off) = *reinterpret_cast<const U *>(s_rec + off);
            };
            copy(trx_a4_kcode<HD>(p, l), uint32_t());
            copy(trx_a4_vcode<HD>(p, l, 0), uint16_t());
            copy(trx_a4_vcode<HD>(p, l, 1), uint16_t());
            if ((l & 3) == 0) {
                copy(Y::KD + trx_a4_flat<HD>(p, g), uint16_t());
                copy(Y::KM + trx_a4_flat<HD>(p, g), uint16_t());
                copy(Y::VD + trx_a4_pair<HD>(p, g), uint16_t());
                copy(Y::VM + trx_a4_pair<HD>(p, g), uint16_t());
            }
        }
    }
    float l1 = 0.0f, h1 = 0.0f;
    if (tid < HD) {
        l1 = s_lo[0][tid], h1 = s_hi[0][tid];
#pragma unroll
        for (int r = 1; r < 8; r++) l1 = fminf(l1, s_lo[r][tid]), h1 = fmaxf(h1, s_hi[r][tid]);
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
        int8_t *o = a.bounds + at * (2 * HD) + tid;
        o[0] = bad ? 0 : (int8_t)fmaxf(floorf(__fmul_rn(l1, per)), -127.0f);
        o[HD] = bad ? 0 : (int8_t)fminf(ceilf(__fmul_rn(h1, per)), 127.0f);
        if (tid == 0) a.units[at] = bad ? INFINITY : unit;
    }
}

// The rows of an entry's block read back (the write's grid), by way of shared memory; a lane 16 bytes of a row, so that a
// warp writes 512 contiguous bytes. Bound by HBM: 4096 rows of 16 heads of 128 (f32, 77 MB) 11.6 us, the measured copy rate
// (by 32 bytes a lane 20.5 us).
template <int HD, typename T>
__global__ void __launch_bounds__(256) trx_a4_read(TrxA4 a, TrxA4Batch b, T *__restrict__ k, int64_t k_stride,
                                                   T *__restrict__ v, int64_t v_stride) {
    constexpr int PER = 16 / sizeof(T), L = HD / PER, ROWS = 256 / L;
    __shared__ __align__(16) uint8_t s_rec[TrxA4L<HD>::BLOCK];
    int slot, row0, rows, pos0;
    const int tid = threadIdx.x, kv = blockIdx.y;
    if (!trx_a4_entry(a, b, blockIdx.z, slot, row0, rows, pos0)) return;
    const int blk = pos0 / TRX_A4_BLOCK + blockIdx.x, first = blk * TRX_A4_BLOCK;
    if (first >= pos0 + rows) return;
    const uint8_t *rec = a.cache + (((int64_t)slot * a.n_kv + kv) * a.n_blocks + blk) * TrxA4L<HD>::BLOCK;
    for (int i = tid; i < TrxA4L<HD>::BLOCK / 16; i += 256)
        reinterpret_cast<uint4 *>(s_rec)[i] = reinterpret_cast<const uint4 *>(rec)[i];
    __syncthreads();
    const int p0 = max(pos0, first) - first, p1 = min(pos0 + rows - first, TRX_A4_BLOCK), l = tid % L;
    for (int p = p0 + tid / L; p < p1; p += ROWS) {
        const int64_t row = row0 + (first + p - pos0);
        T *kr = k + row * k_stride + kv * HD + PER * l, *vr = v + row * v_stride + kv * HD + PER * l;
        if constexpr (PER == 8) {
            float x[8];
            trx_a4_key8<HD>(s_rec, p, l, x);
            trx_a4_store8(kr, x);
            trx_a4_value8<HD>(s_rec, p, l, x);
            trx_a4_store8(vr, x);
        } else {
            float4 x;
            float d, m;
            trx_a4_key_scale<HD>(s_rec, p, l >> 3, d, m);
            trx_a4_value4(*reinterpret_cast<const uint16_t *>(s_rec + trx_a4_kcode<HD>(p, l >> 1) + 2 * (l & 1)), d, m, &x.x);
            *reinterpret_cast<float4 *>(kr) = x;
            trx_a4_value_scale<HD>(s_rec, p, l >> 3, d, m);
            trx_a4_value4(*reinterpret_cast<const uint16_t *>(s_rec + trx_a4_vcode<HD>(p, l >> 1, l & 1)), d, m, &x.x);
            *reinterpret_cast<float4 *>(vr) = x;
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Attention.
//
// With the query x = q 2^-e of a row, a key's score is scale 2^e sum_g (d_g sum_i x_gi c_gi + m_g sum_i x_gi), and an
// output group is (sum_t (p_t d_tg) c_tg + sum_t p_t m_tg) / sum_t p_t: the codes go into the tensor cores as they
// are, and scales and minima are applied to a 32nd of the values.
//
// Codes as f16: four bits masked out of a word (c or 16 c in each half) are an f16 subnormal, c 2^-24 or 16 c 2^-24,
// exactly: a word of 8 codes is one shift and four ANDs, and no subtraction of a bias. The query values that meet a
// 16 c are stored divided by 16; the outputs that come of one are divided by 16 at the end, where 2^24 goes too.
//
// A warp takes records of 32 positions through its own ring of two, 16 positions at a time. (It fills the ring with
// 16-byte asynchronous copies, a group a record: a bulk copy, which one lane issues, held the warp up for 600 of 2800
// cycles a record.)
//   scores   mma m16n8k16: A = 16 keys x 16 codes, B = 8 query rows (f32 rows: a second B with what f16 drops of the
//            first); a group is two of them, then d; the minima's sums are one m16n8k8 with B = sum_i x_gi in two f16
//            parts
//   softmax  a reference a row, which moves only when a score passes it (16-bit rows: by 2^8), so that the usual record
//            needs one vote and no reduction; p in f16 (f32 rows: two f16 parts, 22 bits), transposed in registers (movmatrix).
//            16-bit rows' p, p d and subnormal codes leave f16 outputs 6.5e-4 off 64 bits at 131,000 positions of random values,
//            whose outputs' own rounding is 2e-4 (bf16: 1.6e-3, nearly all of it the outputs'); codes as integers 3.4e-4 at
//            100,000, for a third more time
//   outputs  mma m16n8k16: A = 16 dims x 16 positions of codes, B = p_t d_tg of 8 rows; one more with the minima (and
//            ones, which sum p) as A.
// 16 query rows of f16 or bf16 type, or 8 (R), share the codes' unpacking; scores, sums and outputs are f32.
// p stays below 2^15 / max(1, d): the reference that is subtracted in the exponent is the row's maximum so far, plus
// the binary logarithm of the largest value scale so far where it is above 1, less a constant. Where all scales so far are
// below 2^-8 they are multiplied up to 1: without it, values of 3e-5 behind a position of 2^16 times their weight came out
// 3e-2 off.
//
// A cluster of CTAs shares one tile of query rows: its warps take records in turn, their results are joined in each
// CTA through shared memory, and the CTAs' through distributed shared memory, so that no workspace or second launch is
// needed and overlapping calls share nothing.
//
// What bounds it: HBM where the CTAs fill the GPU (64 sequences of 8192 positions, 32 heads over 8 of 128, bf16: 115 us, 5.8
// TB/s, 0.89 of the measured copy rate); a record's 454 warp instructions where clusters leave SMs idle (one such sequence of
// 131,072 positions: 47.5 us, 3.5 TB/s on 80 SMs) or many rows share the records (f32 prompts).
#define TRX_A4_STAGES 2

__device__ __forceinline__ void trx_a4_mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void trx_a4_mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0));
}
// an 8 x 8 matrix of f16 pairs (lane: row l / 4, columns 2 (l % 4), + 1), transposed
__device__ __forceinline__ uint32_t trx_a4_transpose(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ trx_f2 trx_fma2(trx_f2 a, trx_f2 b, trx_f2 c) {
    trx_f2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
// 2^x within 2^-22 (relative), 0 for -inf
__device__ __forceinline__ float trx_a4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t trx_a4_half2(float lo, float hi) { return trx_a4_pack2(lo, hi, (const __half *)nullptr); }
__device__ __forceinline__ float2 trx_a4_float2(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2 *>(&h)); }
__device__ __forceinline__ uint32_t trx_a4_hmul2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t trx_a4_hadd2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint32_t trx_a4_hfms2(uint32_t a, uint32_t b, uint32_t c) { // a b - c
    uint32_t d;
    asm("{\n .reg .b32 t;\n neg.f16x2 t, %3;\n fma.rn.f16x2 %0, %1, %2, t;\n}" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t trx_a4_hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
// a pair of scales, the NaN among them as 0
__device__ __forceinline__ uint32_t trx_a4_finite(uint32_t d) {
    return ((d & 0xffffu) > 0x7c00u ? 0u : d & 0xffffu) | ((d >> 16) > 0x7c00u ? 0u : d & 0xffff0000u);
}
// NW consecutive words of shared memory
template <int NW> __device__ __forceinline__ void trx_a4_lds(const uint8_t *p, uint32_t (&w)[NW]) {
    if constexpr (NW == 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (NW == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x, w[1] = v.y;
    } else w[0] = *reinterpret_cast<const uint32_t *>(p);
}

__device__ __forceinline__ uint32_t trx_a4_cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void trx_a4_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
// the address of CTA rank's copy of a shared variable, in the cluster's window
__device__ __forceinline__ uint32_t trx_a4_peer(const void *p, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(trx_smem(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ float4 trx_a4_peer_load4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ float trx_a4_peer_load(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}

template <int HD, int R, int W> struct TrxA4Tile { // shared memory of a tile of R query rows, CTAs of W warps
    static constexpr int RING = W * TRX_A4_STAGES * TrxA4L<HD>::REC, PARTS = W * R * (HD + 2) * 4;
    static constexpr int PART = RING > PARTS ? RING : PARTS; // the ring, then in its place the warps' results
    static constexpr int SMEM = PART + R * (HD + 2) * 4;     // behind them the CTA's result
};

// A call's query and output rows: rows of type f32 (F32), else bf16 or f16
struct TrxA4Rows {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    int bf16;
};
template <bool F32> __device__ __forceinline__ void trx_a4_q8(const TrxA4Rows &io, int64_t at, float (&x)[8]) {
    if constexpr (F32) trx_a4_load8((const float *)io.q + at, x);
    else if (io.bf16) trx_a4_load8((const __nv_bfloat16 *)io.q + at, x);
    else trx_a4_load8((const __half *)io.q + at, x);
}
template <bool F32> __device__ __forceinline__ float trx_a4_q1(const TrxA4Rows &io, int64_t at) {
    if constexpr (F32) return ((const float *)io.q)[at];
    const uint16_t u = ((const uint16_t *)io.q)[at];
    return io.bf16 ? trx_bf16(u) : trx_half(u);
}
template <bool F32> __device__ __forceinline__ void trx_a4_out4(const TrxA4Rows &io, int64_t at, float4 v) {
    if constexpr (F32) *reinterpret_cast<float4 *>((float *)io.out + at) = v;
    else if (io.bf16)
        *reinterpret_cast<uint2 *>((__nv_bfloat16 *)io.out + at) =
            make_uint2(trx_a4_pack2(v.x, v.y, (const __nv_bfloat16 *)nullptr), trx_a4_pack2(v.z, v.w, (const __nv_bfloat16 *)nullptr));
    else
        *reinterpret_cast<uint2 *>((__half *)io.out + at) = make_uint2(trx_a4_half2(v.x, v.y), trx_a4_half2(v.z, v.w));
}

// The codes at bits 0 and 4 of a word's halves as two pairs of f16: the integers themselves less MID (EXACT), or c 2^-24
// and 16 c 2^-24. (A word's other four: of the word shifted by 8.)
template <bool EXACT, int MID = 0> __device__ __forceinline__ void trx_a4_half_codes(uint32_t w, uint32_t (&h)[2]) {
    static_assert(MID == 0 || MID == 8, "");
    if constexpr (EXACT) { // 1024 + c and 1024 + 16 c from their bits
        constexpr uint32_t a = MID ? 0xe408e408u : 0xe400e400u, b = MID ? 0xd480d480u : 0xd400d400u; // -1024 - MID, -64 - MID
        h[0] = trx_a4_hadd2((w & 0x000f000fu) | 0x64006400u, a);
        h[1] = trx_a4_hfma2((w & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, b);
    } else {
        h[0] = w & 0x000f000fu, h[1] = w & 0x00f000f0u;
    }
}
template <bool EXACT, int MID = 0> __device__ __forceinline__ void trx_a4_codes(uint32_t w, uint32_t (&h)[4]) {
    uint32_t a[2], b[2];
    trx_a4_half_codes<EXACT, MID>(w, a);
    trx_a4_half_codes<EXACT, MID>(w >> 8, b);
    h[0] = a[0], h[1] = a[1], h[2] = b[0], h[3] = b[1];
}

__device__ __forceinline__ void trx_a4_add4(float (&a)[4], const float (&b)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        trx_f2 x = trx_pack2(a[i], a[i + 1]);
        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(trx_pack2(b[i], b[i + 1])));
        a[i] = trx_lo(x), a[i + 1] = trx_hi(x);
    }
}

// One warp's state for R query rows: NT tiles of 8
template <int HD, bool F32, int R> struct TrxA4Warp {
    // f32 rows take the codes as integers, the values' around their middle: the codes' sums and the minima's would else be
    // far larger than what they leave, and the tensor core's additions do not round (subnormal codes lose 3 to 10 bits
    // more in them, which 16-bit rows can spare)
    static constexpr bool EXACT = F32;
    static constexpr int MID = F32 ? 8 : 0;
    static constexpr int NG = HD / 32, NT = R / 8, NB = F32 ? 2 : NT;
    static_assert(R == 8 || (R == 16 && !F32), "8 rows, or 16 of a 16-bit type");
    // scores of 16-bit types may pass the reference by 2^LAZY before the sums are rescaled
    static constexpr float LAZY = F32 ? 0.0f : 8.0f, TOP = F32 ? 14.0f : 7.0f;
    static constexpr float NONE = -3.0e38f; // the maximum of a row that has seen no position
    uint32_t qb[NB][2 * NG][2]; // the query fragments: lane (n = lane / 4, c = lane % 4) has row n (+ 8)
    uint32_t qs[NT];            // their groups' sums
    int lim[NT];                // the last position row n (+ 8) sees; -1: no row
    float c[NT][2];             // rows 2 c, 2 c + 1 (+ 8): the scores' factor, with log2(e),
    float top[NT][2], ref[NT][2]; // the running maximum, and what the exponent subtracts
    // 2^ed = edlim is above the largest value scale so far: from 2^-8 on at least 1, and the references take it up; below,
    // scales are multiplied by 2^-ed (small values' products with p would be among f16's smallest numbers, or 0)
    int ed;
    float edlim;
    float acc[NG][2][NT][4], accm[NT][4];

    // the query rows of the tile: row r of it is at off(r); rows past n_rows are zero
    template <typename Off>
    __device__ __forceinline__ void load(const TrxA4Rows &io, int lane, int n_rows, float scale, Off off) {
        const int n = lane >> 2, cc = lane & 3;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const bool on = n + 8 * t < n_rows;
            const int64_t at = on ? off(n + 8 * t) : 0;
            float x[NG][8], most = 0.0f, sum[NG];
            bool bad = false;
#pragma unroll
            for (int g = 0; g < NG; g++) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[g][j] = 0.0f;
                if (on) trx_a4_q8<F32>(io, at + 32 * g + 8 * cc, x[g]);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    most = fmaxf(most, fabsf(x[g][j]));
                    bad |= !(fabsf(x[g][j]) <= 3.402823466e38f);
                }
            }
#pragma unroll
            for (int s = 1; s <= 2; s <<= 1) {
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
                bad |= __shfl_xor_sync(0xffffffffu, (int)bad, s) != 0;
            }
            // x = q 2^(10 - ex), below 2^10: a group's sum is below 2^15
            int ex = 0;
            if (!bad && most > 0.0f) ex = max((int)((__float_as_uint(most) >> 23) & 255) - 126, -100);
            const float f = __int_as_float((10 - ex + 127) << 23) * (scale < 0.0f ? -1.0f : 1.0f);
            // (in two steps, as 2^(ex + 14) may pass 32 bits: 2^24, where the codes are subnormals; capped, so that a score
            // of 0 stays 0)
            float factor = fminf(fabsf(scale) * (1.44269504088896341f * __int_as_float((ex - 10 + 127) << 23)) *
                                     (EXACT ? 1.0f : 16777216.0f), 3.0e38f);
            if (bad || !(fabsf(scale) <= 3.402823466e38f)) factor = __int_as_float(0x7fffffff);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                c[t][i] = __shfl_sync(0xffffffffu, factor, 4 * (2 * cc + i));
                top[t][i] = ref[t][i] = NONE;
            }
#pragma unroll
            for (int g = 0; g < NG; g++) {
                sum[g] = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[g][j] = bad ? 0.0f : x[g][j] * f;
                    sum[g] += x[g][j];
                    if (!EXACT && (j & 1)) x[g][j] *= 0.0625f;
                }
#pragma unroll
                for (int s = 1; s <= 2; s <<= 1) sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], s);
                // (fragment register, its two dims): (0: 0, 4) (1: 1, 5) of the first k16, (0: 2, 6) (1: 3, 7) of the second
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int o = 0; o < 2; o++) {
                        const float lo = x[g][2 * h + o], hi = x[g][2 * h + o + 4];
                        const uint32_t w = trx_a4_half2(lo, hi);
                        qb[F32 ? 0 : t][2 * g + h][o] = w;
                        if constexpr (F32) {
                            const float2 b = trx_a4_float2(w);
                            qb[1][2 * g + h][o] = trx_a4_half2(lo - b.x, hi - b.y);
                        }
                    }
            }
            uint32_t w[4];
#pragma unroll
            for (int g = 0; g < NG; g += 2) {
                w[g / 2] = trx_a4_half2(sum[g], sum[g + 1]);
                const float2 b = trx_a4_float2(w[g / 2]);
                w[NG / 2 + g / 2] = trx_a4_half2(sum[g] - b.x, sum[g + 1] - b.y);
            }
            if constexpr (NG == 4) qs[t] = cc == 0 ? w[0] : cc == 1 ? w[1] : cc == 2 ? w[2] : w[3];
            else qs[t] = cc == 0 ? w[0] : cc == 1 ? w[1] : 0u;
#pragma unroll
            for (int i = 0; i < 4; i++) accm[t][i] = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[g][h][t][i] = 0.0f;
        }
        ed = -15, edlim = 3.0517578125e-5f;
    }

    // one record (32 positions from pos0); MASK: some row does not see all of them
    template <bool MASK> __device__ __forceinline__ void record(uint8_t *rec, int lane, int pos0) {
        using L = TrxA4L<HD>;
        const int n = lane >> 2, cc = lane & 3;
        float s[2][NT][4]; // 16 positions each: n (0, 1) and n + 8 (2, 3) x rows 2 cc, 2 cc + 1
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint8_t *p0 = rec + (16 * t + n) * (HD / 2) + cc * (NG * 4);
            const uint8_t *ps = rec + L::KD + (16 * t + n) * (NG * 2);
            uint32_t w0[NG], w1[NG], d0[NG / 2], d1[NG / 2], m[2];
            trx_a4_lds<NG>(p0, w0);
            trx_a4_lds<NG>(p0 + 8 * (HD / 2), w1);
            trx_a4_lds<NG / 2>(ps, d0);
            trx_a4_lds<NG / 2>(ps + 8 * (NG * 2), d1);
#pragma unroll
            for (int k = 0; k < 2; k++)
                m[k] = *reinterpret_cast<const uint32_t *>(ps + (L::KM - L::KD) + 8 * k * (NG * 2) + (NG == 4 ? (cc & 1) * 4 : 0));
            trx_f2 a[NT][2];
#pragma unroll
            for (int r = 0; r < NT; r++) {
                float e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                trx_a4_mma8(e, m[0], m[1], qs[r]);
                a[r][0] = trx_pack2(e[0], e[1]), a[r][1] = trx_pack2(e[2], e[3]);
                if constexpr (!EXACT) {
                    const trx_f2 tiny = trx_pack2(5.9604644775390625e-8f, 5.9604644775390625e-8f); // 2^-24
                    a[r][0] = trx_mul2(a[r][0], tiny), a[r][1] = trx_mul2(a[r][1], tiny);
                }
            }
            // (the groups' products side by side: each waits for the one before it in its group only)
            float x[NG][NT][4];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    uint32_t u[2], v[2];
                    trx_a4_half_codes<EXACT>(h ? w0[g] >> 8 : w0[g], u);
                    trx_a4_half_codes<EXACT>(h ? w1[g] >> 8 : w1[g], v);
#pragma unroll
                    for (int r = 0; r < NT; r++) {
                        if (h == 0) x[g][r][0] = x[g][r][1] = x[g][r][2] = x[g][r][3] = 0.0f;
#pragma unroll
                        for (int b = r; b < NB; b += NT)
                            trx_a4_mma16(x[g][r], u[0], v[0], u[1], v[1], qb[b][2 * g + h][0], qb[b][2 * g + h][1]);
                    }
                }
#pragma unroll
            for (int g = 0; g < NG; g++) {
                const float2 e0 = trx_a4_float2(d0[g / 2]), e1 = trx_a4_float2(d1[g / 2]);
                const float f0 = g & 1 ? e0.y : e0.x, f1 = g & 1 ? e1.y : e1.x;
#pragma unroll
                for (int r = 0; r < NT; r++) {
                    a[r][0] = trx_fma2(trx_pack2(x[g][r][0], x[g][r][1]), trx_pack2(f0, f0), a[r][0]);
                    a[r][1] = trx_fma2(trx_pack2(x[g][r][2], x[g][r][3]), trx_pack2(f1, f1), a[r][1]);
                }
            }
#pragma unroll
            for (int r = 0; r < NT; r++) {
                s[t][r][0] = trx_lo(a[r][0]), s[t][r][1] = trx_hi(a[r][0]);
                s[t][r][2] = trx_lo(a[r][1]), s[t][r][3] = trx_hi(a[r][1]);
            }
        }
        // does a score pass its row's reference, or a value scale the largest before?
        uint32_t vd[NG / 2];
        trx_a4_lds<NG / 2>(rec + L::VD + lane * (NG * 2), vd);
        float2 e = trx_a4_float2(vd[0]);
        float big = fmaxf(e.x, e.y);
        if constexpr (NG == 4) {
            e = trx_a4_float2(vd[NG / 2 - 1]);
            big = fmaxf(big, fmaxf(e.x, e.y));
        }
        bool grow = big > edlim;
        float f[NT][2];
#pragma unroll
        for (int r = 0; r < NT; r++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int last = MASK ? __shfl_sync(0xffffffffu, lim[r], 4 * (2 * cc + i)) : 0;
                float best = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        float &x = s[t][r][2 * k + i];
                        x *= c[r][i];
                        if (MASK && pos0 + 16 * t + 8 * k + n > last) x = -INFINITY;
                        best = fmaxf(best, x);
                    }
                // (rounded down, as the reference is rounded up: p must not pass f16 where scores of 2^25 and more lie apart)
                grow |= best > __fadd_rd(top[r][i], LAZY);
                f[r][i] = best;
            }
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int x = 1; x <= 16; x <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
            float units = 1.0f; // the outputs' by the scales' multiplier
            if (big > edlim) {
                const int x = (int)((__float_as_uint(big) >> 23) & 255) - 126, was = ed; // 2^x > big
                ed = x > -8 ? max(x, 0) : x;
                edlim = __int_as_float((ed + 127) << 23);
                if (was < 0) units = __int_as_float((was - min(ed, 0) + 127) << 23);
            }
#pragma unroll
            for (int r = 0; r < NT; r++) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
#pragma unroll
                    for (int x = 4; x <= 16; x <<= 1) f[r][i] = fmaxf(f[r][i], __shfl_xor_sync(0xffffffffu, f[r][i], x));
                    top[r][i] = fmaxf(top[r][i], f[r][i]);
                    const float to = top[r][i] == NONE ? NONE : __fadd_ru(top[r][i], (float)max(ed, 0) - TOP);
                    f[r][i] = ref[r][i] == to ? 1.0f : trx_a4_exp2(ref[r][i] - to);
                    ref[r][i] = to;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) accm[r][i] *= f[r][i & 1];
                f[r][0] *= units, f[r][1] *= units;
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[g][h][r][i] *= f[r][i & 1];
            }
        }
        float mid = (float)MID;
        if (ed < 0) { // (the record is this warp's until it is fetched over)
#pragma unroll
            for (int k = 0; k < NG / 2; k++)
                *reinterpret_cast<uint32_t *>(rec + L::VD + lane * (NG * 2) + 4 * k) =
                    trx_a4_hmul2(vd[k], (uint32_t)(15 - ed) * 0x04000400u);
            mid = __int_as_float((ed + 127) << 23) * (float)MID;
            __syncwarp();
        }
        uint32_t ps[4][NT], pls[4]; // 8 positions each
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int r = 0; r < NT; r++) {
                const float x = trx_a4_exp2(s[k / 2][r][2 * (k & 1)] - ref[r][0]), y = trx_a4_exp2(s[k / 2][r][2 * (k & 1) + 1] - ref[r][1]);
                const uint32_t h = trx_a4_half2(x, y);
                ps[k][r] = trx_a4_transpose(h);
                if constexpr (F32) {
                    const float2 b = trx_a4_float2(h);
                    pls[k] = trx_a4_transpose(trx_a4_half2(x - b.x, y - b.y));
                }
            }
#pragma unroll
        for (int t = 0; t < 2; t++) { // 16 positions: two tiles of 8
            uint32_t w[2][NG], d[2][NG], m[2], ml[2] = {0u, 0u}, ok[2][NT];
            const uint32_t(&p)[2][NT] = reinterpret_cast<const uint32_t(&)[2][NT]>(ps[2 * t]);
            const uint32_t(&pl)[2] = reinterpret_cast<const uint32_t(&)[2]>(pls[2 * t]);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                trx_a4_lds<NG>(rec + L::V + (2 * t + k) * (4 * HD) + lane * (NG * 4), w[k]);
                trx_a4_lds<NG>(rec + L::VD + (8 * t + 4 * k + cc) * (NG * 4), d[k]);
                // rows 0 .. NG - 1 of A are the groups' minima, row NG ones
                m[k] = n < NG ? *reinterpret_cast<const uint32_t *>(rec + L::VM + (8 * t + 4 * k + cc) * (NG * 4) + n * 4)
                              : n == NG ? 0x3c003c00u : 0u;
                // (m + 8 d) / 16, which f16 holds for every m and d, and (rows n + 8) what 16 times its rounding drops: no
                // smaller than f16's smallest numbers, of which m and 8 d are multiples; a NaN belongs to every row where
                // all see the position
                if constexpr (MID != 0) {
                    const uint32_t x = n < NG ? *reinterpret_cast<const uint32_t *>(rec + L::VD + (8 * t + 4 * k + cc) * (NG * 4) + n * 4) : 0u;
                    const float2 md = trx_a4_float2(m[k]), dd = trx_a4_float2(MASK ? trx_a4_finite(x) : x);
                    const float y = __fmaf_rn(dd.x, mid, md.x), z = __fmaf_rn(dd.y, mid, md.y);
                    m[k] = trx_a4_half2(y * 0.0625f, z * 0.0625f);
                    const float2 r = trx_a4_float2(m[k]);
                    ml[k] = trx_a4_half2(__fmaf_rn(r.x, -16.0f, y), __fmaf_rn(r.y, -16.0f, z));
                }
#pragma unroll
                for (int r = 0; r < NT; r++) {
                    // (a masked position's scale may be a NaN)
                    if constexpr (MASK) {
                        const int at = pos0 + 16 * t + 8 * k + 2 * cc;
                        ok[k][r] = (at <= lim[r] ? 0xffffu : 0u) | (at + 1 <= lim[r] ? 0xffff0000u : 0u);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < NT; r++) {
                float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                float(&o)[4] = F32 ? y : accm[r];
                if constexpr (F32) trx_a4_mma16(o, m[0], ml[0], m[1], ml[1], pl[0], pl[1]);
                trx_a4_mma16(o, m[0], ml[0], m[1], ml[1], p[0][r], p[1][r]);
                if constexpr (F32) trx_a4_add4(accm[r], y);
            }
#pragma unroll
            for (int g = 0; g < NG; g++) {
                uint32_t u[4], v[4];
                trx_a4_codes<EXACT, MID>(w[0][g], u);
                trx_a4_codes<EXACT, MID>(w[1][g], v);
#pragma unroll
                for (int r = 0; r < NT; r++) {
                    uint32_t b0 = trx_a4_hmul2(p[0][r], d[0][g]), b1 = trx_a4_hmul2(p[1][r], d[1][g]);
                    // (f32: 16 positions from 0, then added with rounding: the tensor core's additions to a sum do not round,
                    // and 131,072 positions of 8 KV heads were 7.6e-6 off 64 bits, now about 1e-6, for 6 to 8 % of the time.
                    // 16-bit rows: no change beside their roundings of p)
                    float y[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
                    float(&o0)[4] = F32 ? y[0] : acc[g][0][r], (&o1)[4] = F32 ? y[1] : acc[g][1][r];
                    if constexpr (F32) { // p d in two parts: what the product's rounding drops, and the lower part's product
                        uint32_t l0 = trx_a4_hfma2(pl[0], d[0][g], trx_a4_hfms2(p[0][r], d[0][g], b0));
                        uint32_t l1 = trx_a4_hfma2(pl[1], d[1][g], trx_a4_hfms2(p[1][r], d[1][g], b1));
                        if constexpr (MASK) l0 &= ok[0][r], l1 &= ok[1][r];
                        trx_a4_mma16(o0, u[0], u[1], v[0], v[1], l0, l1);
                        trx_a4_mma16(o1, u[2], u[3], v[2], v[3], l0, l1);
                    }
                    if constexpr (MASK) b0 &= ok[0][r], b1 &= ok[1][r];
                    trx_a4_mma16(o0, u[0], u[1], v[0], v[1], b0, b1);
                    trx_a4_mma16(o1, u[2], u[3], v[2], v[3], b0, b1);
                    if constexpr (F32) trx_a4_add4(acc[g][0][r], y[0]), trx_a4_add4(acc[g][1][r], y[1]);
                }
            }
        }
    }

    // this warp's rows into o [R][HD] (not yet divided) with their references and sums
    __device__ __forceinline__ void store(int lane, float *o, float *refs, float *sums) {
        const int n = lane >> 2, cc = lane & 3;
#pragma unroll
        for (int r = 0; r < NT; r++)
#pragma unroll
            for (int i = 0; i < 2; i++) { // query row 2 cc + i
                const int row = 8 * r + 2 * cc + i;
                if (n == 0) refs[row] = ref[r][i];
                const float own = MID ? __fmaf_rn(accm[r][i], 16.0f, accm[r][2 + i]) : accm[r][i]; // a group's minima, or ones
                if (n == NG) sums[row] = own;
#pragma unroll
                for (int g = 0; g < NG; g++) { // dims 32 g + 4 n + 0..3
                    const float m = __shfl_sync(0xffffffffu, own, 4 * g + cc);
                    const float x = __int_as_float((min(ed, 0) + 127) << 23);
                    const float e = (EXACT ? 1.0f : 16777216.0f) * x, f = (EXACT ? 1.0f : 1048576.0f) * x; // 2^24, 2^20
                    *reinterpret_cast<float4 *>(o + row * HD + 32 * g + 4 * n) =
                        make_float4(__fmaf_rn(acc[g][0][r][i], e, m), __fmaf_rn(acc[g][0][r][2 + i], f, m),
                                    __fmaf_rn(acc[g][1][r][i], e, m), __fmaf_rn(acc[g][1][r][2 + i], f, m));
                }
            }
    }
};

// A tile of query rows (row r: its values at off_q(r) and off_o(r), its last position lim(r)) over the first n_units
// records (of the listed blocks, or 0, 1, ..), by the CTAs of the cluster (ranks of them). smem: TrxA4Tile::SMEM bytes,
// 128-byte aligned; what was read of it is ordered before (the caller's barrier).
template <int HD, bool F32, int R, int W, typename Lim, typename OffQ, typename OffO>
__device__ __forceinline__ void trx_a4_tile(uint8_t *smem, const TrxA4Rows &io, const uint8_t *recs,
                                            const int *list, int n_units, int n_rows, int last, float scale, int ranks,
                                            Lim lim, OffQ off_q, OffO off_o) {
    constexpr int REC = TrxA4L<HD>::REC, S = TRX_A4_STAGES;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = ranks > 1 ? (int)trx_a4_cluster_rank() : 0;
    if (n_units <= W) { // one CTA's work: the others leave, and nobody meets
        if (rank > 0) return;
        ranks = 1;
    }
    uint8_t *ring = smem + warp * (S * REC);
    const int step = ranks * W;
    auto record = [&](int u) { return list ? 2 * list[u >> 1] + (u & 1) : u; }; // the u-th record's index
    auto fetch = [&](int u, int st) {
        if (u < n_units) {
            const uint8_t *src = recs + (int64_t)record(u) * REC + lane * 16;
            const uint32_t dst = trx_smem(ring + st * REC + lane * 16);
#pragma unroll
            for (int i = 0; i < REC / 512; i++)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + i * 512), "l"(src + i * 512) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int u = rank * W + warp;
#pragma unroll
    for (int i = 0; i < S; i++) fetch(u + i * step, i);
    TrxA4Warp<HD, F32, R> w;
    w.load(io, lane, n_rows, scale, off_q);
    int low = last; // the lowest of the rows' last positions
#pragma unroll
    for (int t = 0; t < R / 8; t++) {
        const int r = (lane >> 2) + 8 * t;
        w.lim[t] = r < n_rows ? lim(r) : -1;
        if (r < n_rows) low = min(low, w.lim[t]);
    }
    low = __reduce_min_sync(0xffffffffu, low) - (TRX_A4_REC - 1);
    for (int st = 0; u < n_units; u += step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(TRX_A4_STAGES - 1) : "memory");
        __syncwarp();
        const int pos = record(u) * TRX_A4_REC;
        if (pos <= low) w.template record<false>(ring + st * REC, lane, pos);
        else w.template record<true>(ring + st * REC, lane, pos);
        __syncwarp();
        fetch(u + S * step, st);
        st = st + 1 == S ? 0 : st + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads(); // the rings are free
    float *o = reinterpret_cast<float *>(smem), *refs = o + W * R * HD, *sums = refs + W * R;
    float *co = reinterpret_cast<float *>(smem + TrxA4Tile<HD, R, W>::PART), *cref = co + R * HD, *csum = cref + R;
    w.store(lane, o + warp * R * HD, refs + warp * R, sums + warp * R);
    __syncthreads();
    constexpr int ITEMS = R * HD / 4;
    for (int x = tid; x < ITEMS; x += 32 * W) { // the CTA's warps joined, in their order
        const int r = x / (HD / 4), d = x % (HD / 4) * 4;
        float top = refs[r];
#pragma unroll
        for (int k = 1; k < W; k++) top = fmaxf(top, refs[k * R + r]);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < W; k++) {
            const float f = trx_a4_exp2(refs[k * R + r] - top);
            const float4 y = *reinterpret_cast<const float4 *>(o + (k * R + r) * HD + d);
            sum = __fmaf_rn(f, sums[k * R + r], sum);
            v = make_float4(__fmaf_rn(f, y.x, v.x), __fmaf_rn(f, y.y, v.y), __fmaf_rn(f, y.z, v.z), __fmaf_rn(f, y.w, v.w));
        }
        if (ranks == 1) {
            if (r < n_rows)
                trx_a4_out4<F32>(io, off_o(r) + d, make_float4(__fdiv_rn(v.x, sum), __fdiv_rn(v.y, sum),
                                                               __fdiv_rn(v.z, sum), __fdiv_rn(v.w, sum)));
        } else {
            *reinterpret_cast<float4 *>(co + r * HD + d) = v;
            if (d == 0) cref[r] = top, csum[r] = sum;
        }
    }
    if (ranks == 1) return;
    trx_a4_cluster_sync();
    // the CTAs joined: CTA rank takes an even share of the values, `lanes` neighbouring lanes (a power of two) one of them
    const int lanes = ranks <= 2 ? 2 : ranks <= 4 ? 4 : ranks <= 8 ? 8 : 16;
    const int share = (ITEMS + ranks - 1) / ranks, k = tid % lanes, peer = min(k, ranks - 1);
    for (int j0 = 0; j0 < share; j0 += 32 * W / lanes) {
        const int j = j0 + tid / lanes, i = min(rank * share + j, ITEMS - 1), r = i / (HD / 4), d = i % (HD / 4) * 4;
        const float own = trx_a4_peer_load(trx_a4_peer(cref + r, peer));
        float sum = trx_a4_peer_load(trx_a4_peer(csum + r, peer));
        float4 v = trx_a4_peer_load4(trx_a4_peer(co + r * HD + d, peer));
        float top = own;
        for (int x = 1; x < lanes; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float f = trx_a4_exp2(own - top);
        const bool on = k < ranks; // (a lane without a CTA adds nothing)
        sum = on ? sum * f : 0.0f;
        v = on ? make_float4(v.x * f, v.y * f, v.z * f, v.w * f) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int x = 1; x < lanes; x <<= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, x);
            v.x += __shfl_xor_sync(0xffffffffu, v.x, x);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, x);
            v.z += __shfl_xor_sync(0xffffffffu, v.z, x);
            v.w += __shfl_xor_sync(0xffffffffu, v.w, x);
        }
        if (k == 0 && j < share && rank * share + j < ITEMS && r < n_rows)
            trx_a4_out4<F32>(io, off_o(r) + d, make_float4(__fdiv_rn(v.x, sum), __fdiv_rn(v.y, sum),
                                                           __fdiv_rn(v.z, sum), __fdiv_rn(v.w, sum)));
    }
    trx_a4_cluster_sync(); // no CTA leaves while another reads its memory
}

// The entry a CTA takes in a call of more CTAs than fit at once: the blockIdx.z-th longest, so that the shortest are left
// for the end (n_entries <= the CTA's threads, all of which call)
template <int W> __device__ __forceinline__ int trx_a4_longest(const TrxA4Batch &b, int z) {
    __shared__ __align__(16) int s_len[32 * W];
    __shared__ int s_entry;
    const int i = threadIdx.x, n = b.n_entries;
    int len = 0;
    if (i < n && b.slot[i] >= 0) len = b.pos0[i] + (b.start ? b.start[i + 1] - b.start[i] : 1);
    s_len[i] = i < n ? len : INT_MIN;
    __syncthreads();
    int before = 0;
    for (int j = 0; j < n; j += 4) {
        const int4 x = *reinterpret_cast<const int4 *>(s_len + j);
        before += (x.x > len || (x.x == len && j < i)) + (x.y > len || (x.y == len && j + 1 < i)) +
                  (x.z > len || (x.z == len && j + 2 < i)) + (x.w > len || (x.w == len && j + 3 < i));
    }
    if (i < n && before == z) s_entry = i;
    __syncthreads();
    return s_entry;
}

// blockIdx.x = tile of R rows (token-major, a KV head's query heads side by side; the last tiles, whose contexts are the
// longest, first) x KV head x CTA of the cluster, z the entry
template <int HD, bool F32, int R, int W>
__global__ void __launch_bounds__(32 * W, R == 8 ? 16 / W : 1)
    trx_a4_attend(TrxA4 a, TrxA4Batch b, TrxA4Rows io, float scale, int ranks, int sorted) {
    extern __shared__ __align__(128) uint8_t smem[];
    int slot, row0, rows, pos0;
    const int kv = blockIdx.x / ranks % a.n_kv, G = a.n_head / a.n_kv;
    const int entry = sorted ? trx_a4_longest<W>(b, blockIdx.z) : blockIdx.z;
    if (!trx_a4_entry(a, b, entry, slot, row0, rows, pos0)) return;
    const int total = rows * G, tiles = (total + R - 1) / R, tile = tiles - 1 - (int)(blockIdx.x / ranks / a.n_kv);
    if (tile < 0) return;
    const uint8_t *recs = a.cache + ((int64_t)slot * a.n_kv + kv) * a.n_blocks * TrxA4L<HD>::BLOCK;
    const int r0 = tile * R, n_rows = min(R, total - r0), last = pos0 + (r0 + n_rows - 1) / G;
    auto at = [&](int64_t stride, int r) {
        const int x = r0 + r, tok = x / G;
        return (int64_t)(row0 + tok) * stride + (int64_t)(kv * G + x - tok * G) * HD;
    };
    trx_a4_tile<HD, F32, R, W>(
        smem, io, recs, nullptr, last / TRX_A4_REC + 1, n_rows, last, scale, ranks,
        [&](int r) { return pos0 + (r0 + r) / G; }, [&](int r) { return at(io.q_stride, r); },
        [&](int r) { return at(io.out_stride, r); });
}

// a float as an unsigned key of the same order (no NaN)
__device__ __forceinline__ uint32_t trx_a4_key(float f) {
    const uint32_t u = __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Attention to n_sel blocks: the row's own and the n_sel - 1 earlier ones of the best scores (ties to the lowest
// index). A block's score is f32(sum_i P_i highest_i + N_i lowest_i) x unit, what the group's summed q.k can reach (up to
// the roundings) in whole numbers: P_i and N_i sum the positive and the negative parts of the group's query values, which are rounded
// to multiples of a power of two that puts the largest magnitude in [64, 128) and kept within 127. Sums of whole
// numbers do not depend on their order, so neither does the selection. A block with a NaN among its keys scores +inf;
// a query with one selects by index. blocks (optional): the selected blocks, ascending, then -1.
//
// A cluster shares a (row, KV head): each CTA scores an even part of the earlier blocks (a warp a block: 2 HD bytes, dp2a,
// one warp reduction) and keeps the keys in shared memory; the threshold is found 8 bits at a time from the CTAs' joined
// histograms; each CTA sends its selected blocks to every CTA's list, and the cluster attends to the list.
// blockIdx.x = (row x tiles of R heads) x CTA of the cluster, y the KV head, z the entry. Dynamic shared memory: the
// tile's (the keys take its place before it starts), at least keys x 4 bytes, then n_sel ints (list_at).
// What bounds it: latency. 24 x 4 rows, 16 of up to 512 blocks, 16 heads of 64 over 4, f32: 36 us in 1.3 rounds of CTAs, of
// whose 34,500 cycles 10 % load the queries, 24 % score, 16 % find the threshold, 5 % make the list, 45 % attend. One row,
// 32 of 2047 blocks, 32 heads over 8 of 128, bf16: 17 us (all positions 48).
template <int HD, bool F32, int R, int W>
__global__ void __launch_bounds__(32 * W, R == 8 ? 16 / W : 1)
    trx_a4_select(TrxA4 a, TrxA4Batch b, TrxA4Rows io, float scale, int n_sel, int32_t *__restrict__ blocks, int ranks,
                  int list_at) {
    constexpr int N = 32 * W, PW = HD / 64; // words of bounds a lane takes of a block
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(16) int16_t s_pn[2 * HD]; // N, then P, as the bounds (read as words)
    __shared__ int s_hist[4][256], s_warp[2][W], s_cnt[2], s_pick[2][3], s_before[2];
    int slot, row0, rows, pos0;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kv = blockIdx.y, G = a.n_head / a.n_kv;
    const int tiles = (G + R - 1) / R, r = (int)(blockIdx.x / ranks) / tiles, h0 = (int)(blockIdx.x / ranks) % tiles * R;
    if (!trx_a4_entry(a, b, blockIdx.z, slot, row0, rows, pos0) || r >= rows) return;
    const int rank = (int)trx_a4_cluster_rank();
    const int pos = pos0 + r, home = pos / TRX_A4_BLOCK, n_list = min(home + 1, n_sel);
    const int64_t at = ((int64_t)slot * a.n_kv + kv) * a.n_blocks;
    const int64_t qr = (int64_t)(row0 + r) * io.q_stride + (int64_t)kv * G * HD;
    uint32_t *s_key = reinterpret_cast<uint32_t *>(smem);
    int *list = reinterpret_cast<int *>(smem + list_at);
    if (home + 1 > n_sel && n_sel > 1) {
        float most = 0.0f;
        int bad = 0;
        for (int i = tid; i < G * HD; i += N) {
            const float f = fabsf(trx_a4_q1<F32>(io, qr + i));
            bad |= !(f <= 3.402823466e38f);
            most = fmaxf(most, f);
        }
        for (int i = tid; i < 4 * 256; i += N) (&s_hist[0][0])[i] = 0;
        for (int s = 16; s; s >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
        if (lane == 0) s_warp[0][warp] = __float_as_int(most);
        bad = __syncthreads_or(bad);
        most = 0.0f;
        for (int i = 0; i < W; i++) most = fmaxf(most, __int_as_float(s_warp[0][i]));
        if (tid < HD) {
            int ex = 0, up = 0, down = 0;
            if (most > 0.0f && !bad) frexpf(most, &ex);
            for (int h = 0; h < G; h++) {
                const float f = trx_a4_q1<F32>(io, qr + h * HD + tid);
                const int z = bad ? 0 : (int)fminf(fmaxf(rintf(ldexpf(f, 7 - ex)), -127.0f), 127.0f);
                up += max(z, 0);
                down += min(z, 0);
            }
            s_pn[tid] = (int16_t)down, s_pn[HD + tid] = (int16_t)up;
        }
        __syncthreads();
        const int per = (home + ranks - 1) / ranks, base = rank * per, cnt = max(0, min(per, home - base));
        int pn[2 * PW];
#pragma unroll
        for (int i = 0; i < 2 * PW; i++) pn[i] = reinterpret_cast<const int *>(s_pn)[lane * (2 * PW) + i];
        const int8_t *bounds = a.bounds + (at + base) * (2 * HD);
        constexpr int F = 8; // blocks a step; the next step's are on their way
        int w[2][F][PW];
        auto look = [&](int (&x)[F][PW], int g) {
            const int8_t *p = bounds + (int64_t)g * (2 * HD) + lane * (4 * PW);
#pragma unroll
            for (int i = 0; i < F; i++) {
                const bool on = g + i < cnt;
                if constexpr (PW == 2) {
                    const int2 v = on ? *reinterpret_cast<const int2 *>(p + i * (2 * HD)) : make_int2(0, 0);
                    x[i][0] = v.x, x[i][1] = v.y;
                } else x[i][0] = on ? *reinterpret_cast<const int *>(p + i * (2 * HD)) : 0;
            }
        };
        auto score = [&](const int (&x)[F][PW], int g) {
            int mine = 0;
            float u = 0.0f;
            if (lane < F && g + lane < cnt) u = a.units[at + base + g + lane];
#pragma unroll
            for (int i = 0; i < F; i++) {
                int sum = 0;
#pragma unroll
                for (int k = 0; k < PW; k++) sum = __dp2a_hi(pn[2 * k + 1], x[i][k], __dp2a_lo(pn[2 * k], x[i][k], sum));
                sum = __reduce_add_sync(0xffffffffu, sum);
                if (lane == i) mine = sum;
            }
            if (lane < F && g + lane < cnt) s_key[g + lane] = trx_a4_key(u == INFINITY ? INFINITY : __fmul_rn((float)mine, u));
        };
        look(w[0], warp * F);
#pragma unroll 1
        for (int g = warp * F; g < cnt; g += 2 * W * F) {
            look(w[1], g + W * F);
            score(w[0], g);
            look(w[0], g + 2 * W * F);
            score(w[1], g + W * F);
        }
        __syncthreads();
        // the largest key that at least n_sel - 1 blocks reach, and how many of the blocks at that key are taken
        uint32_t key = 0;
        int want = n_sel - 1;
        auto meet = [&] {
            if (ranks > 1) trx_a4_cluster_sync();
            else __syncthreads();
        };
        bool all = false; // the last bin's blocks are all taken: the key's other bits do not matter
        for (int pass = 0; pass < 4 && !all; pass++) {
            const int shift = 24 - 8 * pass;
            const uint32_t mask = pass == 0 ? 0u : 0xffffffffu << (shift + 8);
            for (int i0 = 0; i0 < cnt; i0 += N) {
                const int i = i0 + tid;
                const bool on = i < cnt && (s_key[i] & mask) == key;
                const uint32_t bin = on ? (s_key[i] >> shift) & 255u : 256u;
                const uint32_t same = __match_any_sync(0xffffffffu, bin); // (most keys share their first bits)
                if (on && lane == __ffs(same) - 1) atomicAdd(&s_hist[pass][bin], __popc(same));
            }
            meet();
            int n = 0; // thread: a bin (of 256)
            if (ranks == 1) n = s_hist[pass][tid];
            else
                for (int k = 0; k < ranks; k++) n += __float_as_int(trx_a4_peer_load(trx_a4_peer(&s_hist[pass][tid], k)));
            int above = n; // its blocks and those of the higher bins
            for (int s = 1; s < 32; s <<= 1) {
                const int x = __shfl_down_sync(0xffffffffu, above, s);
                if (lane + s < 32) above += x;
            }
            if (lane == 0) s_warp[0][warp] = above;
            __syncthreads();
            for (int i = warp + 1; i < W; i++) above += s_warp[0][i];
            if (above >= want && above - n < want) s_pick[pass & 1][0] = tid, s_pick[pass & 1][1] = want - (above - n), s_pick[pass & 1][2] = n;
            __syncthreads();
            key |= (uint32_t)s_pick[pass & 1][0] << shift;
            want = s_pick[pass & 1][1];
            all = want == s_pick[pass & 1][2] && key > 0;
        }
        if (all) key--, want = 0;
        // this CTA's blocks above the key and at it, and those of the CTAs before
        int place = 0, ties = 0;
        if (ranks > 1) {
            int above = 0, equal = 0;
            for (int i = tid; i < cnt; i += N) above += s_key[i] > key, equal += s_key[i] == key;
            above = __reduce_add_sync(0xffffffffu, above);
            equal = __reduce_add_sync(0xffffffffu, equal);
            if (lane == 0) s_warp[0][warp] = above, s_warp[1][warp] = equal;
            __syncthreads();
            if (tid < 2) {
                int n = 0;
                for (int i = 0; i < W; i++) n += s_warp[tid][i];
                s_cnt[tid] = n;
            }
            trx_a4_cluster_sync();
            if (tid == 0) {
                int eq = 0, n = 0;
                for (int k = 0; k < rank; k++) {
                    n += __float_as_int(trx_a4_peer_load(trx_a4_peer(&s_cnt[0], k)));
                    eq += __float_as_int(trx_a4_peer_load(trx_a4_peer(&s_cnt[1], k)));
                }
                s_before[0] = n + min(eq, want), s_before[1] = eq;
            }
            __syncthreads();
            place = s_before[0], ties = s_before[1];
        }
        for (int i0 = 0; i0 < cnt; i0 += N) { // ascending
            const int i = i0 + tid;
            const bool eq = i < cnt && s_key[i] == key;
            const uint32_t e = __ballot_sync(0xffffffffu, eq);
            if (lane == 0) s_warp[1][warp] = __popc(e);
            __syncthreads();
            int before = ties, all = ties;
            for (int x = 0; x < W; x++) {
                if (x < warp) before += s_warp[1][x];
                all += s_warp[1][x];
            }
            const bool take = (i < cnt && s_key[i] > key) || (eq && before + __popc(e & ((1u << lane) - 1)) < want);
            const uint32_t t = __ballot_sync(0xffffffffu, take);
            if (lane == 0) s_warp[0][warp] = __popc(t);
            __syncthreads();
            int to = place;
            for (int x = 0; x < W; x++) {
                if (x < warp) to += s_warp[0][x];
                place += s_warp[0][x];
            }
            ties = all;
            if (take) {
                to += __popc(t & ((1u << lane) - 1));
                if (ranks == 1) list[to] = i;
                else
                    for (int k = 0; k < ranks; k++)
                        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(trx_a4_peer(list + to, k)), "r"(base + i) : "memory");
            }
            __syncthreads();
        }
        if (tid == 0) list[n_sel - 1] = home;
        meet();
    } else {
        for (int i = tid; i < n_list; i += N) list[i] = n_sel == 1 ? home : i;
    }
    __syncthreads(); // (the keys' place becomes the ring)
    if (blocks && h0 == 0 && rank == 0)
        for (int i = tid; i < n_sel; i += N)
            blocks[((int64_t)(row0 + r) * a.n_kv + kv) * n_sel + i] = i < n_list ? list[i] : -1;
    const uint8_t *recs = a.cache + at * TrxA4L<HD>::BLOCK;
    const int64_t outr = (int64_t)(row0 + r) * io.out_stride + (int64_t)kv * G * HD;
    trx_a4_tile<HD, F32, R, W>(
        smem, io, recs, list, 2 * (n_list - 1) + (pos % TRX_A4_BLOCK) / TRX_A4_REC + 1, min(R, G - h0), pos, scale,
        ranks, [&](int) { return pos; }, [&](int x) { return qr + (h0 + x) * HD; }, [&](int x) { return outr + (h0 + x) * HD; });
}
