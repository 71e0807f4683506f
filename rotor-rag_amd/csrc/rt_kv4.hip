// A KV cache held in 4 bits: RoPE + quantising append, read-back, and causal GQA attention
// over it, for B sequences that each stand at a position of their own.
//
// Callers in the reference: MultiHeadAttention.forward (src/rotor/transformer.py:206-292: KV
// concat :250-252, GQA repeat :260-263, scores/softmax/AV :267-281) with the per-layer cache
// list of BitNetModel.forward (src/rotor/bitnet_model.py:223-228); its cache is fp32.
//
// A group is 64 consecutive dimensions of one head at one position: codes c = 0..15 and two
// bf16 numbers, the middle z and the half step h; value = z + h (2 c - 15).
//
// A layer's cache is [B][Hkv][ceil(Lmax / 64) blocks], a block being 64 positions of one head,
// in dwords:
//   K codes   [64 positions][4 h][HD/64 g][2 e]: dimensions 64 g + 16 h + 8 e + (0..7)
//   V codes   [HD/32 u][16 d][4 = 2 s + l][2 v][2 w]: dimension 32 u + 16 v + d, positions
//             32 w + 16 s + 4 l + (0, 1, 2, 3, 8, 9, 10, 11)
//   K scales  [HD/64][64 positions]: z << 16 | h;   V scales the same
// Element e of a dword's eight lies in nibble e / 2 + 4 (e % 2).  Codes lie as the matrix
// instructions take them: lane (i = l % 16, h = l / 16) of a 16x16x32 product loads 16 bytes
// of a key (its 8 (2) dimensions of each of the products over d) or 16 bytes of a value dimension (its
// 8 keys of two products for two dimension tiles), every byte of the block once and in order.
// The keys of a dword are those that the scores' products leave in one lane (register r of
// lane group h holds row 4 h + r), so the softmax's numbers are the value products' operand
// as they are.
//
// Floating-point contraction is off: what is rounded where is part of the cache's definition.
#include <algorithm>
#include <type_traits>

#include "rt_internal.h"

#pragma clang fp contract(off)

namespace rt {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kKv4Block = 64;  // positions in a block

__host__ __device__ constexpr int kv4_block_bytes(int hd) { return 72 * hd; }

// Shift of element e in a dword of eight codes.
__device__ __forceinline__ int kv4_shift(int e) { return 4 * (e >> 1) + 16 * (e & 1); }

__device__ __forceinline__ unsigned bf16_bits(float x) {  // x finite or infinite: round to nearest even
    const unsigned u = __float_as_uint(x);
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ float kv4_z(unsigned s) { return __uint_as_float(s & 0xFFFF0000u); }
__device__ __forceinline__ float kv4_h(unsigned s) { return __uint_as_float(s << 16); }

// z and h of a group from its extremes, as the cache's dword.  By definition in 64 bits up to the
// roundings, so that nothing hangs on the order of fp32 operations.  z in fp32 is the same number; h
// in fp32 is within 2^-22 of it, so its bf16 is the same unless it lies next to a border: those (one
// group in 2000) and very small ones take the division.  A group with a value that is not finite, or
// whose z or h is not, reads as NaN.
__device__ __forceinline__ unsigned kv4_scale(float lo, float hi, bool finite) {
    float fz = 0.5f * hi + 0.5f * lo, fh = (0.5f * hi - 0.5f * lo) * (1.0f / 15.0f);
    const unsigned low = __float_as_uint(fh) & 0xFFFFu;
    if (low - 0x7FF0u <= 0x20u || !(fabsf(fh) >= 0x1p-90f) || !(fabsf(fh) <= 0x1p100f)) {
        const double a = 0.5 * (double)lo, b = 0.5 * (double)hi;
        fz = (float)(b + a);
        fh = (float)((b - a) / 15.0);
    }
    const unsigned z = bf16_bits(fz), h = bf16_bits(fh);
    const bool ok = finite && (z & 0x7F80u) != 0x7F80u && (h & 0x7F80u) != 0x7F80u;
    return ok ? z << 16 | h : 0x7FC00000u;
}
// The codes of eight values.  In fp32, ((x - z) / h + 15) / 2 is off by less than 2^-18: only where it
// lies within 2^-16 of a border (or is no number: h = 0, or too small for its reciprocal) is the
// definition's 64-bit form needed, one element in 30000.
__device__ __forceinline__ unsigned kv4_encode(const float (&x)[8], unsigned s) {
    const float z = kv4_z(s), h = kv4_h(s), inv = 1.0f / h;
    float c[8];
    bool close = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float y = ((x[e] - z) * inv + 15.0f) * 0.5f;
        c[e] = rintf(y);
        close = close || !(fabsf(y - c[e]) <= 0.5f - 0x1p-16f);
    }
    if (close) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double t = h == 0.0f ? 0.0 : ((double)x[e] - (double)z) / (double)h;
            c[e] = (float)rint((t + 15.0) * 0.5);
        }
    }
    unsigned w = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= (unsigned)(int)fminf(fmaxf(c[e], 0.0f), 15.0f) << kv4_shift(e);
    return w;
}

// Scale dword (s) and codes of a group whose 64 numbers eight neighbour lanes hold, eight each.
__device__ __forceinline__ unsigned kv4_group(const float (&x)[8], int lane, unsigned& s) {
    float lo = x[0], hi = x[0];
    bool fin = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
        fin = fin && fabsf(x[e]) <= 3.402823466e38f;
    }
#pragma unroll
    for (int w = 1; w < 8; w <<= 1) {
        lo = fminf(lo, __shfl_xor(lo, w, 64));
        hi = fmaxf(hi, __shfl_xor(hi, w, 64));
    }
    const unsigned long long bad = __ballot(!fin);
    s = kv4_scale(lo, hi, ((bad >> (lane & 56)) & 0xFFull) == 0ull);
    return kv4_encode(x, s);
}
// Dimensions 8 o .. 8 o + 7 of a key at p, rotated (src: the head's row).
template <int HD>
__device__ __forceinline__ void kv4_rotate(float (&x)[8], const float* src, const float* rope, int p, int o) {
    constexpr int HALF = HD / 2;
    const bool up = 8 * o >= HALF;
    const int i = (8 * o) % HALF;
    const float* other = src + (up ? i : i + HALF);
    const float* cs = rope + ((size_t)p * HALF + i) * 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const double a = x[e], d = other[e], c = cs[2 * e], s = cs[2 * e + 1];
        x[e] = up ? (float)(a * c + d * s) : (float)(a * c - d * s);
    }
}
// Where a block keeps the codes of 8 dimensions of a key, and the eight values' dword of a dimension
// (positions 16 x + 4 vl + (0..3, 8..11)) at p.
template <int HD>
__device__ __forceinline__ int kv4_key_word(int p, int o) {
    return p % kKv4Block * (HD / 8) + (o % 8 / 2) * (HD / 32) + o / 8 * 2 + o % 2;
}
template <int HD>
__device__ __forceinline__ int kv4_value_word(int p, int vl, int dim) {
    return 8 * HD + ((dim / 32 * 16 + dim % 16) * 4 + p % 32 / 16 * 2 + vl) * 4 + dim % 32 / 16 * 2 + p % kKv4Block / 32;
}

// A row (b, m) stands at position pos[b] + m; rows outside [0, Lmax) have no place in the cache.
__device__ __forceinline__ int kv4_row_pos(int pos, int m, int Lmax) {
    const long long p = (long long)pos + m;
    return p >= 0 && p < Lmax ? (int)p : -1;
}

// ---- append ------------------------------------------------------------------------------
// Workgroups [0, nkv): 16 positions of one KV head of one sequence (the positions whose codes
// share dwords of V); threads 0..127 take K, 128..255 V, each thread 8 dimensions of a position,
// the 8 threads of a group finding its extremes by exchange.  V's codes go through LDS into
// dwords; a dword with positions outside this call keeps their nibbles.  The rest: 4 pairs of
// a query a thread.
// RoPE in 64 bits, rounded once: the products are exact there, so every order gives this value.
constexpr int kKv4Rows = 16;

template <int HD>
__global__ void __launch_bounds__(256) kv4_append_kernel(const float* q, const float* __restrict__ k,
                                                         const float* __restrict__ v, const float* __restrict__ rope,
                                                         uint8_t* __restrict__ cache, float* q_out, int B, int M,
                                                         int H, int Hkv, int Lmax, int nblk, int chunks, int nkv,
                                                         const int* __restrict__ pos_p) {
    constexpr int HALF = HD / 2, TPR = HD / 8;  // threads a row
    __shared__ unsigned codes[kKv4Rows][TPR];
    const int t = threadIdx.x;
    if ((int)blockIdx.x >= nkv) {
        const long long idx = (long long)((int)blockIdx.x - nkv) * 256 + t;
        const int i = (int)(idx % (HALF / 4)) * 4;
        const long long hr = idx / (HALF / 4);  // (row, head)
        const long long row = hr / H;
        if (row >= (long long)B * M) return;
        const int b = (int)(row / M), m = (int)(row % M), p = kv4_row_pos(pos_p[b], m, Lmax);
        const v4f x1 = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(q + hr * HD + i));
        const v4f x2 = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(q + hr * HD + HALF + i));
        v4f y1{}, y2{};
        if (p >= 0) {
            const v4f cs0 = *reinterpret_cast<const v4f*>(rope + ((size_t)p * HALF + i) * 2);
            const v4f cs1 = *reinterpret_cast<const v4f*>(rope + ((size_t)p * HALF + i) * 2 + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double c = j < 2 ? cs0[2 * j] : cs1[2 * j - 4], s = j < 2 ? cs0[2 * j + 1] : cs1[2 * j - 3];
                y1[j] = (float)((double)x1[j] * c - (double)x2[j] * s);
                y2[j] = (float)((double)x2[j] * c + (double)x1[j] * s);
            }
        }
        *reinterpret_cast<v4f*>(q_out + hr * HD + i) = y1;
        *reinterpret_cast<v4f*>(q_out + hr * HD + HALF + i) = y2;
        return;
    }
    const int chunk = blockIdx.x % chunks, bh = blockIdx.x / chunks, b = bh / Hkv, kh = bh % Hkv;
    const int pos = pos_p[b];
    const long long first = (long long)max(pos, 0) / kKv4Rows * kKv4Rows + (long long)chunk * kKv4Rows;
    const long long end = min((long long)pos + M, (long long)Lmax);  // positions [pos, end) are this call's
    if (first >= end) return;  // (uniform over the workgroup)
    const int p0 = (int)first, lane = t & 63;
    uint8_t* const blk = cache + ((size_t)bh * nblk + p0 / kKv4Block) * kv4_block_bytes(HD);
    const bool is_v = t >= 128;
    const int o = t % TPR;  // dimensions 8 o .. 8 o + 7
    unsigned* const sc = reinterpret_cast<unsigned*>(blk + 64 * HD) + (is_v ? HD : 0);
    // V's dword of thread (dimension, l): positions 4 l + (0..3, 8..11) of the 16; what it holds is asked for
    // now, for the positions that are not this call's
    const int dim = min(t >> 1, HD - 1), vl = t & 1;
    unsigned* const vat = reinterpret_cast<unsigned*>(blk) + kv4_value_word<HD>(p0, vl, dim);
    const unsigned old = pos > p0 || end < first + kKv4Rows ? *vat : 0u;
    for (int r0 = 0; r0 < kKv4Rows; r0 += 128 / TPR) {
        if (p0 + r0 >= end || p0 + r0 + 128 / TPR <= pos) continue;  // (uniform) none of these rows
        const int r = r0 + (t & 127) / TPR, p = p0 + r;
        const bool in = p >= pos && p < end;
        float x[8];
        const float* src = (is_v ? v : k) + ((size_t)b * M + (in ? p - pos : 0)) * Hkv * HD + (size_t)kh * HD;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = src[8 * o + e];
        if (!is_v) kv4_rotate<HD>(x, src, rope, in ? p : 0, o);
        unsigned s;
        const unsigned word = kv4_group(x, lane, s);
        const int P = p % kKv4Block;
        if (is_v) codes[r][o] = word;
        if (in) {
            if (!is_v) reinterpret_cast<unsigned*>(blk)[kv4_key_word<HD>(p, o)] = word;
            if (o % 8 == 0) sc[o / 8 * 64 + P] = s;
        }
    }
    __syncthreads();
    if (t >= 2 * HD) return;
    unsigned word = 0u, keep = 0xFFFFFFFFu;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int r = 8 * (e >> 2) + 4 * vl + (e & 3), p = p0 + r;
        if (p >= pos && p < end) {
            word |= ((codes[r][dim / 8] >> kv4_shift(dim % 8)) & 15u) << kv4_shift(e);
            keep &= ~(15u << kv4_shift(e));
        }
    }
    if (keep != 0xFFFFFFFFu) *vat = (old & keep) | word;
}

// ---- read --------------------------------------------------------------------------------
// Rows (b, m) of K and V as fp32 [B][Hkv][M][HD].  A workgroup takes the rows of one block of 64
// positions of one head (blocks in front of the cache and behind it too: zeros).  A thread has 4
// dimensions of 8 positions (4 at 64 dimensions), so that every store instruction writes whole rows:
// with a position and a dimension a thread it was stores of 4 bytes, 4 x 32768 positions (5 heads of
// 128) 440 us.
template <int HD>
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint8_t* __restrict__ cache, float* __restrict__ k,
                                                       float* __restrict__ v, int M, int Hkv, int Lmax, int nblk,
                                                       int chunks, const int* __restrict__ pos_p) {
    constexpr int LR = HD / 4, N = 64 * LR / 256;  // lanes a row, positions a thread
    const int chunk = blockIdx.x % chunks, bh = blockIdx.x / chunks, t = threadIdx.x;
    const int pos = pos_p[bh / Hkv], grp = t / LR, d = t % LR * 4, g = d / 64;
    const long long j = (pos >> 6) + (long long)chunk;  // (rounds down)
    if (j * kKv4Block >= (long long)pos + M) return;
    const bool in = j >= 0 && j < nblk;
    const uint8_t* blk = cache + ((size_t)bh * nblk + (in ? j : 0)) * kv4_block_bytes(HD);
    const unsigned *w = reinterpret_cast<const unsigned*>(blk), *sc = w + 16 * HD + g * 64;
    // K: positions N grp + n.  V: the N positions from number first_v on of the eight of dword (w, s, l) = octet
    const int octet = grp * N / 8, first_v = grp * N % 8, vbase = 32 * (octet >> 2) + 16 * (octet >> 1 & 1) + 4 * (octet & 1);
    // rows of this call: number m, -1 for none
    auto row = [&](int P) {
        const long long m = j * kKv4Block + P - pos;
        return m >= 0 && m < M ? (int)m : -1;
    };
    unsigned kw[N], ks[N], vw[4], vs[N];
    bool any = false;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int P = N * grp + n, e = first_v + n, Pv = vbase + 8 * (e >> 2) + (e & 3);
        const bool kin = in && row(P) >= 0, vin = in && row(Pv) >= 0;
        kw[n] = kin ? w[P * (HD / 8) + d % 64 / 16 * (HD / 32) + g * 2 + d % 16 / 8] : 0u;
        ks[n] = kin ? sc[P] : 0u;
        vs[n] = vin ? sc[HD + Pv] : 0u;
        any = any || vin;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
        vw[c] = any ? w[8 * HD + ((d / 32 * 16 + (d + c) % 16) * 4 + (octet & 3)) * 4 + d % 32 / 16 * 2 + (octet >> 2)] : 0u;
    const size_t base = (size_t)bh * M * HD + d;
    auto put = [&](float* out, int P, const v4f& x) {
        const int m = row(P);
        const long long p = j * kKv4Block + P;
        if (m >= 0) __builtin_nontemporal_store(p >= 0 && p < Lmax ? x : v4f{}, reinterpret_cast<v4f*>(out + base + (size_t)m * HD));
    };
#pragma unroll
    for (int n = 0; n < N; ++n) {
        v4f x;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            x[c] = kv4_z(ks[n]) + kv4_h(ks[n]) * (float)(2 * (int)((kw[n] >> kv4_shift(d % 8 + c)) & 15u) - 15);
        put(k, N * grp + n, x);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int e = first_v + n;
        v4f x;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            x[c] = kv4_z(vs[n]) + kv4_h(vs[n]) * (float)(2 * (int)((vw[c] >> kv4_shift(e)) & 15u) - 15);
        put(v, vbase + 8 * (e >> 2) + (e & 3), x);
    }
}

// ---- attention ---------------------------------------------------------------------------
// The levels 2 c - 15 of two of a dword's codes, exact in fp16: a nibble at bits 4..7 of a half under
// 0x6400 is 1024 + 16 c, and (1024 + 16 c) / 8 - 143 = 2 c - 15.  Masking and setting the
// exponent are one v_and_or_b32, which takes one of its two constants from a VGPR: `mask` is
// kv4_mask()'s.
__device__ __forceinline__ unsigned kv4_mask(unsigned m = 0x00F000F0u) {
    asm("" : "+v"(m));
    return m;
}
__device__ __forceinline__ v2h kv4_level2(unsigned w, int i, unsigned mask) {  // elements 2 i, 2 i + 1
    const v2h f = {(_Float16)0.125f, (_Float16)0.125f}, o = {(_Float16)-143.0f, (_Float16)-143.0f};
    const unsigned n = i == 0 ? w << 4 : w >> (4 * i - 4);
    return __builtin_elementwise_fma(__builtin_bit_cast(v2h, (n & mask) | 0x64006400u), f, o);
}
// c - 8 for the eight codes of a dword, elements 2, 3, 6 and 7 16 (c - 8): nine instructions instead of
// eleven.  (As fp16 subnormals, c 2^-24, five would do, and the matrix instructions take them, but align
// products by the exponents they would have if normal: results were off by 2^-18.)
__device__ __forceinline__ v8h kv4_codes(unsigned w, unsigned mask, unsigned mask0) {
    const v2h o = {(_Float16)-1032.0f, (_Float16)-1032.0f}, o16 = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const unsigned v = w >> 8;
    const v2h x[4] = {__builtin_bit_cast(v2h, (w & mask0) | 0x64006400u) + o, __builtin_bit_cast(v2h, (w & mask) | 0x64006400u) + o16,
                      __builtin_bit_cast(v2h, (v & mask0) | 0x64006400u) + o, __builtin_bit_cast(v2h, (v & mask) | 0x64006400u) + o16};
    v8h r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[2 * i] = x[i][0];
        r[2 * i + 1] = x[i][1];
    }
    return r;
}
// x (|x| < 2^15) as two fp16 terms: the error is at most 2^-22 |x| or 2^-25.  The empty asm keeps
// the product that x comes from and its conversion apart: fused (v_fma_mixlo_f16) in one use of
// hi and not in the other, hi differs by its last bit in one of some ten thousand, and that
// much of x was lost (5e-6 of a result over 8192 keys).
__device__ __forceinline__ float kv4_minus_one() {
    float m = -1.0f;
    asm("" : "+s"(m));
    return m;
}
__device__ __forceinline__ void kv4_split(float& a, float& b, v2h& hi, v2h& lo) {  // (a and b as they were)
    asm("" : "+v"(a), "+v"(b));
    hi = __builtin_convertvector((v2f{a, b}), v2h);
    // (- 1.0 as a number that the compiler does not see: a subtraction would convert hi first)
    const float m = kv4_minus_one();
    lo = __builtin_convertvector((v2f{fmaf((float)hi[0], m, a), fmaf((float)hi[1], m, b)}), v2h);
}
__device__ __forceinline__ void kv4_split(v2f x, v2h& hi, v2h& lo) {
    float a = x[0], b = x[1];
    kv4_split(a, b, hi, lo);
}
// 2^n as fp32, -126 <= n <= 127
__device__ __forceinline__ float kv4_pow2(int n) { return __uint_as_float((unsigned)(n + 127) << 23); }
__device__ __forceinline__ int kv4_exponent(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 127; }

// Joins the lanes l, l ^ 16, l ^ 32, l ^ 48 (all four get the result); x in two lane halves only.
template <typename Op>
__device__ __forceinline__ float kv4_join32(float x, Op op) {
    const v2u y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
template <typename Op>
__device__ __forceinline__ float kv4_join16(float x, Op op) {
    const v2u y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return kv4_join32(op(__uint_as_float(y[0]), __uint_as_float(y[1])), op);
}
// The largest of a wave's numbers, in an SGPR.
__device__ __forceinline__ unsigned kv4_wave_max(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xF, 0xF, false));  // row_ror 1, 2, 4, 8
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xF, 0xF, false));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xF, 0xF, false));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xF, 0xF, false));
    const v2u y = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(y[0], y[1]);
    const v2u w = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __builtin_amdgcn_readfirstlane(max(w[0], w[1]));
}
// What a wave's lanes wrote to LDS is there for its other lanes: LDS takes a wave's accesses in order, so this is for the
// compiler, and no instruction.
__device__ __forceinline__ void kv4_wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}
struct Kv4Max {
    __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Kv4Min {
    __device__ float operator()(float a, float b) const { return fminf(a, b); }
};
struct Kv4Sum {
    __device__ float operator()(float a, float b) const { return a + b; }
};

struct Kv4AttnArgs {
    const float* q;
    const uint8_t* cache;
    float* out;
    float* work;  // [unit][split] (S = 0: [workgroup]): O [tile rows][HD], (reference, sum of weights) [tile rows][2]
    const int* pos;
    int M, H, Hkv, Lmax, nblk, tiles, S, bh;  // bh = B * Hkv.  S = 0: splits by length (kv4_piece)
    int* heads;                               // S = 0: (pieces, first) of every head
    float scale;  // log2(e) / sqrt(HD)
    // a decode step (M = 1; q not rotated): the new row's key and value, the angles, the cache to write to
    const float *k, *v, *rope;
    uint8_t* put;
};

// What rows m0..m1 of a sequence at pos see: keys [0, kend) some of them, keys [0, all] each of them
// (rows outside the cache see none).
struct Kv4Range {
    int kend, all;
};
__device__ __forceinline__ Kv4Range kv4_range(int pos, int m0, int m1, int Lmax) {
    const long long p0 = (long long)pos + m0, p1 = (long long)pos + m1;
    return {p1 < 0 || p0 >= Lmax ? 0 : (int)min(p1, (long long)Lmax - 1) + 1, p0 < 0 || p1 >= Lmax ? -1 : (int)p0};
}

// Splits by length, for a batch of up to 64 sequences (one tile a unit): with the same number for each, the
// longest decides the launch.  A sequence of n blocks is cut into pieces of at most q of them, q a multiple of
// 4 (a block a wave) for which the pieces of all heads fit the kKv4Slots workgroups that the chip holds at
// once; workgroup w takes pieces in the order (sequence, head, piece).  Every wave works this out for itself,
// lane b for sequence b, and the first piece of a head tells the join where its partials are.
constexpr int kKv4Slots = 512;
struct Kv4Piece {
    int b, head, piece, n, first;  // n pieces a head of sequence b; first: the workgroup of this head's first
};
__device__ __forceinline__ int kv4_wave_scan(int x) {  // inclusive, over the lanes
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15, 31
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return x;
}
// The piece of workgroup w; n = 0: none.
__device__ __forceinline__ Kv4Piece kv4_piece(const Kv4AttnArgs& a, int w, int lane) {
    const int B = a.bh / a.Hkv;
    const int nb = lane < B ? (kv4_range(a.pos[lane], 0, a.M - 1, a.Lmax).kend + kKv4Block - 1) / kKv4Block : 0;
    const long long all = (long long)__builtin_amdgcn_readlane(kv4_wave_scan(nb), 63) * a.Hkv;
    int q = max(4, (int)(all / (kKv4Slots - a.bh / 4) + 3) & ~3), n, incl;
    for (;; q += max(4, q / 16 & ~3)) {  // (ends at the latest with a piece a head: bh <= kKv4Slots)
        n = lane < B ? max(1, (int)(((float)(nb + q - 1) + 0.25f) * (1.0f / (float)q))) : 0;
        incl = kv4_wave_scan(n);
        if (__builtin_amdgcn_readlane(incl, 63) * a.Hkv <= kKv4Slots) break;
    }
    const unsigned long long here = __ballot(w < incl * a.Hkv);
    if (here == 0ull) return Kv4Piece{0, 0, 0, 0, 0};
    Kv4Piece p;
    p.b = (int)__builtin_ctzll(here);
    p.n = __builtin_amdgcn_readlane(n, p.b);
    const int start = (__builtin_amdgcn_readlane(incl, p.b) - p.n) * a.Hkv;
    p.head = (w - start) / p.n;
    p.piece = w - start - p.head * p.n;
    p.first = start + p.head * p.n;
    return p;
}

// The power of two that brings the largest of a row's scaled queries into [2^14, 2^15).
__device__ __forceinline__ int kv4_query_power(float big) { return min(max(14 - kv4_exponent(big), -113), 126); }

// The one new row of a head (k, v: its HD numbers) into its block at p, by one wave, as kv4_append_kernel
// writes it.
template <int HD>
__device__ __forceinline__ void kv4_put_row(const float* k, const float* v, const float* rope, uint8_t* blk, int p, int lane) {
    constexpr int TPR = HD / 8;  // lanes [0, TPR) take the key, the next TPR the value, the rest the value again
    const bool is_v = lane >= TPR;
    const int o = lane % TPR, r = p % 16, vl = r >> 2 & 1, sh = kv4_shift(r >> 3 << 2 | (r & 3));
    unsigned *const words = reinterpret_cast<unsigned*>(blk), *at[HD / 64], old[HD / 64];
#pragma unroll
    for (int n = 0; n < HD / 64; ++n) {
        at[n] = words + kv4_value_word<HD>(p, vl, 64 * n + lane);
        old[n] = *at[n];
    }
    float x[8];
    const float* src = is_v ? v : k;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = src[8 * o + e];
    if (!is_v) kv4_rotate<HD>(x, src, rope, p, o);
    unsigned s;
    const unsigned word = kv4_group(x, lane, s);
    if (!is_v) words[kv4_key_word<HD>(p, o)] = word;
    if (lane < 2 * TPR && o % 8 == 0) words[16 * HD + (is_v ? HD : 0) + o / 8 * 64 + p % kKv4Block] = s;
#pragma unroll
    for (int n = 0; n < HD / 64; ++n) {
        const unsigned w = (unsigned)__shfl((int)word, TPR + 8 * n + lane / 8, 64);
        *at[n] = (old[n] & ~(15u << sh)) | ((w >> kv4_shift(lane % 8)) & 15u) << sh;
    }
    __threadfence_block();  // the wave's loads of the block come after
}
// Rotates queries that lie as the few-rows kernel holds them, with the products and roundings of
// kv4_append_kernel.
template <int HD>
__device__ __forceinline__ void kv4_rotate_query(v4f (&qx)[HD / 64][4], const v4f* cs, int h) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const double co = cs[2 * e + c / 2][2 * (c % 2)], si = cs[2 * e + c / 2][2 * (c % 2) + 1];
            if constexpr (HD == 128) {  // pairs (i, i + 64): both in this lane
                const double a = qx[0][e][c], b = qx[1][e][c];
                qx[0][e][c] = (float)(a * co - b * si);
                qx[1][e][c] = (float)(b * co + a * si);
            } else {  // (i, i + 32): lane groups h and h + 2
                const unsigned u = __float_as_uint(qx[0][e][c]);
                const v2u y = __builtin_amdgcn_permlane32_swap(u, u, false, false);
                const double a = __uint_as_float(y[0]), b = __uint_as_float(y[1]);
                qx[0][e][c] = h < 2 ? (float)(a * co - b * si) : (float)(b * co + a * si);
            }
        }
}

// ---- few rows ------------------------------------------------------------------------------
// A tile is RT rows (R = m G + g of KV head kh), RT = 4, 8 or 16.  The matrix instructions have 16
// columns: column i is row i % RT over the key tiles of number i / RT modulo 16 / RT, so that every
// lane's softmax counts however few the rows (with 16 columns for 4 rows, 12 lanes of 16 worked on
// nothing: 131072 keys, 20 heads over 5, 44 us); the columns of a row are joined at the end.  Lane l
// works on column i = l % 16 with the keys of lane group h = l / 16.  The split's blocks go to its
// NW waves in turn, an online softmax (base 2) for every column:
//   D = C Q^T per group of 64 dimensions (C the keys' codes less 8, exact in fp16; Q two fp16 terms,
//       scaled so that the row's largest is in [2^14, 2^15)),  s = 2 h D + (z + h) sum_d q
//   w = 2^(s - top),  O^T += f C^T (2 w h)^T  (C the values' codes less 8; 2 w h f two fp16 terms),
//       O += sum_j w (z + h)
// so that all products are exact and all sums fp32.  (With c in place of c - 8 the two sums would cancel over
// many keys; with the levels 2 c - 15 themselves a dword takes eleven instructions instead of nine.)  top is the
// largest score so far, and f = 2^(13 - e), 2^e the largest h of the values so far (or 2^-24 of the largest |z|: a
// group's h is no less than 2^-29 of it unless it is 0), which keeps 2 w h f below 2^15.  f is no part of what the
// join sees, nor of the scores' reference: there (top + e - 13, so that one factor served both) it fell to
// rounding beside scores of 2^25 and more, and the references of waves whose values were 2^126 apart did not meet.
// One f for the wave is enough where the steps of its keys' values lie within 2^9 of each other (a row's best key
// then has 2 w h f >= 2^6, and the second fp16 term ends at 2^-25).  From the first block on where they do not,
// or where they are below 2^-80, every column and group of 64 dimensions takes an f of its own, by the largest
// w h that the column has seen (FAR below; a key that it does not see has w = 0): one product a weight and one
// maximum more, and no loads ahead (in every block: 131072 keys, 20 heads over 5, 30.2 us, so 31.5; 512 tokens from an
// empty cache 18.1 / 19.2).  So do waves with a row whose queries' halves differ by more than 2^7: a half's
// largest is then brought into [2^14, 2^15) for itself.
// Every load is issued half a round before its use: the keys of the next block when those of this
// one are multiplied, its values after this one's.  A block's scales are made numbers once, a key a lane,
// and read from LDS by the lanes that use them (each for itself, tiles of 16 rows took 1000 vector
// instructions a block and more registers than there are: 512 / 1024 tokens from an empty cache, 20 heads
// over 5, 20.2 / 40.4 us, so 17.6 / 34.9, with f as above 17.9 / 35; 64 sequences of 4 tokens at 500 17.3, so 13.8).

// A wave's part of a tile of RT rows: blocks j, j + step, .. of head bh.  Column i = lane % 16 (its row, over its key
// tiles) leaves its sums o (dimensions 32 u + 16 v + 4 h + r of o[2 u + v][r]), its largest score and its sum of
// weights.  scales: room for 4 HD floats of the wave's own.  ANY: steps may lie far apart from the first block on.
template <int HD, int RT, bool STEP, bool ANY>
__device__ __forceinline__ void kv4_rows(const Kv4AttnArgs& a, int bh, int tile, int j, int step, float* scales, int lane,
                                         v4f (&o)[HD / 16], float& top, float& lrow) {
    constexpr int NG = HD / 64, NT = HD / 16, NA = 16 / RT, NQ = 4 / NA;  // NQ key tiles of 4 a block are a column's
    const int i = lane & 15, h = lane >> 4, ca = i / RT;
    const int b = bh / a.Hkv, kh = bh % a.Hkv, G = a.H / a.Hkv;
    const unsigned mask = kv4_mask(), mask0 = kv4_mask(0x000F000Fu);
    const int rows = a.M * G, R = min(tile * RT + i % RT, rows - 1), m = R / G;  // (rows past the end repeat the last)
    // the row's queries, dimensions 64 g + 16 h + 8 e + (0..7): requested before the first block, since loads
    // return in order
    v4f qx[NG][4];
    const float* qp = a.q + (((size_t)b * a.M + m) * a.H + (size_t)kh * G + R % G) * HD;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) qx[g][e] = *reinterpret_cast<const v4f*>(qp + 64 * g + 16 * h + 4 * e);
    const int pos = a.pos[b];
    const int last = kv4_row_pos(pos, m, a.Lmax);  // keys <= last are this row's
    const Kv4Range range = kv4_range(pos, tile * RT / G, (min(tile * RT + RT, rows) - 1) / G, a.Lmax);
    const int kend = range.kend, all = range.all;
    const uint8_t* const head = a.cache + (size_t)bh * a.nblk * kv4_block_bytes(HD);
    const int nb = (kend + kKv4Block - 1) / kKv4Block;
    v4f cs[STEP ? 8 : 1];  // cos, sin of pairs 16 (h % (HD / 32)) + (0..15)
    if constexpr (STEP) {
        const float* at = a.rope + ((size_t)max(last, 0) * (HD / 2) + h % (HD / 32) * 16) * 2;
#pragma unroll
        for (int e = 0; e < 8; ++e) cs[e] = *reinterpret_cast<const v4f*>(at + 4 * e);
        const int p = __builtin_amdgcn_readfirstlane(last);
        if (p >= 0 && p / kKv4Block % step == j)
            kv4_put_row<HD>(a.k + (size_t)bh * HD, a.v + (size_t)bh * HD, a.rope,
                            a.put + ((size_t)bh * a.nblk + p / kKv4Block) * kv4_block_bytes(HD), p, lane);
    }
    // Key tile wx = 2 w + x of a block: keys 32 w + 8 x + kl + r of lane group h.  The column's own
    // tiles are wx = NA q + ca.
    const int kl = 16 * (h >> 1) + 4 * (h & 1);
    auto tile_key = [](int wx) { return 32 * (wx >> 1) + 8 * (wx & 1); };
    v4u kc[4], vc[2 * NG];
    unsigned ks[NG], vs[NG];  // scales of key `lane`
    // (byte offsets in a block, whose address is uniform)
    const unsigned at_k = (16 * (i >> 3) + (i & 7)) * (HD / 2) + h * 8 * NG, at_v = 32 * HD + (i * 4 + h) * 16,
                   at_s = 64 * HD + lane * 4;
    auto load_k = [&](int j) {
        const uint8_t* blk = head + (size_t)j * kv4_block_bytes(HD);
#pragma unroll
        for (int wx = 0; wx < 4; ++wx) {
            const uint8_t* kp = blk + (at_k + tile_key(wx) * (HD / 2));
            if constexpr (NG == 2) kc[wx] = *reinterpret_cast<const v4u*>(kp);
            else {
                const v2u x = *reinterpret_cast<const v2u*>(kp);
                kc[wx][0] = x[0];
                kc[wx][1] = x[1];
            }
        }
    };
    auto load_v = [&](int j) {
        const uint8_t* blk = head + (size_t)j * kv4_block_bytes(HD);
#pragma unroll
        for (int u = 0; u < 2 * NG; ++u) vc[u] = *reinterpret_cast<const v4u*>(blk + (at_v + u * 1024));
    };
    auto load_s = [&](int j) {
        const uint8_t* blk = head + (size_t)j * kv4_block_bytes(HD);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            ks[g] = *reinterpret_cast<const unsigned*>(blk + (at_s + 256 * g));
            vs[g] = *reinterpret_cast<const unsigned*>(blk + (at_s + 4 * HD + 256 * g));
        }
    };
    if constexpr (STEP && RT == 16) kv4_rotate_query<HD>(qx, cs, h);  // (no registers for both)
#pragma unroll
    for (int g = 0; g < NG; ++g) ks[g] = vs[g] = 0u;
    if (!ANY && j < nb) {
        load_s(j);
        load_k(j);
        load_v(j);
    }
    if constexpr (STEP && RT != 16) kv4_rotate_query<HD>(qx, cs, h);
    bool far = ANY;
    float zs[NG];
    top = -INFINITY;
    lrow = 0.0f;
    unsigned vmax = 0u;                      // 2^e's number, as bits
    float vmin = INFINITY;                   // the smallest step that the lane has met
    int ve = -110, vn = ve;                  // e of the sums, and with the next block
    int fe[NG];                              // FAR: the columns' f = 2^fe, and
    float seen[NG];                          // the largest 2 w h
    // block j's values' scales, which are loaded: h and z + h as numbers (what lies behind the newest key is not read as
    // one: no step, and where the middle is NaN no row sees it), and with them vmax and vmin (but for groups that
    // read as NaN)
    float vh[NG], vzh[NG];
    auto measure = [&](int j) __attribute__((always_inline)) {
        const bool behind = j * kKv4Block + lane >= kend;
        float big = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float z = behind ? __builtin_nanf("") : kv4_z(vs[g]);
            vh[g] = behind ? 0.0f : kv4_h(vs[g]);
            vzh[g] = z + vh[g];
            big = fmaxf(big, fmaxf(vh[g], fabsf(z) * 0x1p-24f));
            vmin = fminf(vmin, fmaf(z, 0.0f, vh[g]));
        }
        vmax = max(vmax, kv4_wave_max(__float_as_uint(big)));
        vn = max((int)(vmax >> 23) - 127, -110);
        far |= __any(vmin < kv4_pow2(max(vn - 8, -80))) != 0;
    };
    if constexpr (!ANY) measure(j);
    float qs[NG], qi, qr[NG];
    v8h qh[NG][2], ql[NG][2];
    {
        float big[NG], most = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            big[g] = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    qx[g][e][c] *= a.scale;
                    big[g] = fmaxf(big[g], fabsf(qx[g][e][c]));
                }
            big[g] = kv4_join16(big[g], Kv4Max());
            most = fmaxf(most, big[g]);
        }
        const int qe = kv4_query_power(most);
        qi = kv4_pow2(1 - qe);
        // a group that is far smaller than the other has a power of two of its own, which FAR takes off its products
        int dq[NG];
        bool apart = false;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            dq[g] = (int)(NG > 1) & (int)(big[g] > 0.0f) & (int)(most < INFINITY) ? min(kv4_query_power(big[g]) - qe, 126) : 0;
            apart |= __any(dq[g] > 6) != 0;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            dq[g] = apart ? dq[g] : 0;
            const float qf = kv4_pow2(qe + dq[g]);
            qr[g] = kv4_pow2(-dq[g]);
            qs[g] = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                // (every other pair meets codes that are 16 times as large)
                const v2f x = {qx[g][e / 4][e % 4] * qf, qx[g][e / 4][e % 4 + 1] * qf};
                const float part = e & 2 ? 0.0625f : 1.0f;
                v2h hi, lo;
                kv4_split(x * part, hi, lo);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    qh[g][e / 8][e % 8 + c] = hi[c];
                    ql[g][e / 8][e % 8 + c] = lo[c];
                    qs[g] += x[c];
                }
            }
            qs[g] = kv4_join16(qs[g], Kv4Sum()) * (0.5f * qr[g]);
        }
        far |= apart;
    }
    // the block's scales as numbers: h and z + h of the keys, 2 h f and z + h of the values, [64 keys] each, by group
    const v4f* const own_scales = reinterpret_cast<const v4f*>(scales + tile_key(ca) + kl);
    auto scale = [&](int kind, int g, int q) { return own_scales[(64 * (4 * g + kind) + tile_key(NA * q)) / 4]; };
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = v4f{};
#pragma unroll
    for (int g = 0; g < NG; ++g) zs[g] = 0.0f;
    const float two = lane & 2 ? 0.125f : 2.0f;  // (codes 2, 3, 6, 7 come 16 times as large)
    auto walk = [&](auto far_) __attribute__((always_inline)) {
        constexpr bool FAR = decltype(far_)::value;
        for (; j < nb && (FAR || __builtin_expect(!far, 1)); j += step) {
            if constexpr (FAR) {
                load_s(j);
                load_k(j);
                load_v(j);
            }
            const int key0 = j * kKv4Block + kl;
            const bool edge = j * kKv4Block + kKv4Block - 1 > all;  // some row does not see the whole block
            if constexpr (FAR) measure(j);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                scales[64 * (4 * g) + lane] = kv4_h(ks[g]);
                scales[64 * (4 * g + 1) + lane] = kv4_z(ks[g]) + kv4_h(ks[g]);
                scales[64 * (4 * g + 2) + lane] = vh[g] * (two * (FAR ? 1.0f : kv4_pow2(13 - vn)));
                scales[64 * (4 * g + 3) + lane] = vzh[g];
            }
            kv4_wave_lds();
            if (!FAR && j + step < nb) load_s(j + step);
            float s[NQ][4];
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
                v4f own[NG];
#pragma unroll
                for (int c = 0; c < NA; ++c) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        v4f dot{};
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const v8h u = kv4_codes(kc[NA * q + c][2 * g + e], mask, mask0);
                            dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(u, qh[g][e], dot, 0, 0, 0);
                            dot = __builtin_amdgcn_mfma_f32_16x16x32_f16(u, ql[g][e], dot, 0, 0, 0);
                        }
                        if (c == 0) own[g] = dot;
                        else
#pragma unroll
                            for (int r = 0; r < 4; ++r) own[g][r] = ca == c ? dot[r] : own[g][r];
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) s[q][r] = 0.0f;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const v4f kh = scale(0, g, q), kz = scale(1, g, q);
                    if constexpr (FAR && NG > 1) own[g] *= qr[g];
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[q][r] = fmaf(kh[r], own[g][r], fmaf(kz[r], qs[g], s[q][r]));
                }
            }
            if (!FAR && j + step < nb) load_k(j + step);
            if (edge) {
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = key0 + tile_key(NA * q + ca) + r;
                        s[q][r] = key <= last ? s[q][r] : -INFINITY;
                    }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[q][r]);
            const float now = fmaxf(top, kv4_join16(mx, Kv4Max()) * qi);
            if (__any(now != top) || (!FAR && vn != ve)) {
                const float alpha = __builtin_amdgcn_exp2f(top - (now == -INFINITY ? 0.0f : now));
                const float fix = FAR ? alpha : alpha * (ve - vn < -126 ? 0.0f : kv4_pow2(ve - vn));
                lrow *= alpha;
#pragma unroll
                for (int g = 0; g < NG; ++g) zs[g] *= alpha;
                if constexpr (FAR)
#pragma unroll
                    for (int g = 0; g < NG; ++g) seen[g] *= alpha;
#pragma unroll
                for (int n = 0; n < NT; ++n) o[n] *= fix;
                top = now;
                if constexpr (!FAR) ve = vn;
            }
            if constexpr (!FAR) measure(j + step);
            const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[q][r] = __builtin_amdgcn_exp2f(fmaf(s[q][r], qi, -ref));  // (-inf: 0)
                    lrow += s[q][r];
                }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float f = 1.0f;
                if constexpr (FAR) {
                    float big = 0.0f;
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        const v4f wv = scale(2, g, q);
#pragma unroll
                        for (int r = 0; r < 4; ++r) big = fmaxf(big, s[q][r] * wv[r] * (r & 2 ? 16.0f : 1.0f));
                    }
                    seen[g] = fmaxf(seen[g], kv4_join16(big, Kv4Max()));
                    const int n = seen[g] > 0.0f ? min(13 - kv4_exponent(seen[g]), 126) : fe[g];
                    if (__any(n != fe[g])) {
#pragma unroll
                        for (int u = 4 * g; u < 4 * g + 4; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[u][r] = __builtin_ldexpf(o[u][r], n - fe[g]);
                        fe[g] = n;
                    }
                    f = kv4_pow2(n);
                }
                unsigned wh[NQ][2], wl[NQ][2];
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    const v4f wv = scale(2, g, q), vz = scale(3, g, q);
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        v2h hi, lo;
                        kv4_split(v2f{FAR ? s[q][r] * f * wv[r] : s[q][r] * wv[r], FAR ? s[q][r + 1] * f * wv[r + 1] : s[q][r + 1] * wv[r + 1]}, hi, lo);
                        wh[q][r / 2] = __builtin_bit_cast(unsigned, hi);
                        wl[q][r / 2] = __builtin_bit_cast(unsigned, lo);
                    }
                    if (edge) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const bool see = key0 + tile_key(NA * q + ca) + r <= last;
                            zs[g] = fmaf(s[q][r], see ? vz[r] : 0.0f, zs[g]);
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) zs[g] = fmaf(s[q][r], vz[r], zs[g]);
                    }
                }
                // the weights of the products over tiles 2 w and 2 w + 1: the column's own tile, or zeros
                v4u th[2], tl[2];
#pragma unroll
                for (int wx = 0; wx < 4; ++wx)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const bool mine = NA == 1 || wx % NA == ca;
                        th[wx >> 1][2 * (wx & 1) + c] = mine ? wh[wx / NA][c] : 0u;
                        tl[wx >> 1][2 * (wx & 1) + c] = mine ? wl[wx / NA][c] : 0u;
                    }
#pragma unroll
                for (int u = 2 * g; u < 2 * g + 2; ++u)
#pragma unroll
                    for (int v = 0; v < 2; ++v)
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const v8h lev = kv4_codes(vc[u][2 * v + w], mask, mask0);
                            v4f& acc = o[2 * u + v];
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(lev, __builtin_bit_cast(v8h, th[w]), acc, 0, 0, 0);
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(lev, __builtin_bit_cast(v8h, tl[w]), acc, 0, 0, 0);
                        }
            }
            if (!FAR && j + step < nb) load_v(j + step);
            kv4_wave_lds();  // (before the next block's scales)
        }
    };
    if constexpr (!ANY) walk(std::false_type{});
#pragma unroll
    for (int g = 0; g < NG; ++g) fe[g] = ANY ? 0 : 13 - ve;
    if (ANY || __builtin_expect(far && j < nb, 0)) {
#pragma unroll
        for (int g = 0; g < NG; ++g) seen[g] = ANY || top == -INFINITY ? 0.0f : kv4_pow2(ve);
        walk(std::true_type{});
    }
    lrow = kv4_join16(lrow, Kv4Sum());
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        zs[g] = kv4_join16(zs[g], Kv4Sum());
        const float back = kv4_pow2(-fe[g]);
#pragma unroll
        for (int n = 4 * g; n < 4 * g + 4; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[n][r] = fmaf(o[n][r], back, zs[g]);
    }
}

// STEP (one token, G <= 16 so that a head is one tile): append and attention in one launch.  Every
// workgroup rotates its queries; the wave whose block the token lies in writes it there first.
template <int HD, int RT, bool STEP, int NW>
__global__ void __launch_bounds__(64 * NW, 2) kv4_attn_kernel(const Kv4AttnArgs a) {
    constexpr int NT = HD / 16, NA = 16 / RT;
    __shared__ __attribute__((aligned(16))) float om[NW][16][HD + 4];  // (before, each wave's scales of a block)
    __shared__ float ml[NW][16][2];
    const int t = threadIdx.x, lane = t & 63, i = lane & 15, h = lane >> 4;
    int split, S, tile, bh, slot;  // slot: the partial's in the workspace
    if (a.S == 0) {
        const Kv4Piece p = kv4_piece(a, (int)blockIdx.x, lane);
        if (p.n == 0) return;
        split = p.piece;
        S = p.n;
        tile = 0;
        bh = p.b * a.Hkv + p.head;
        slot = p.first + p.piece;
        if (split == 0 && t == 0) {
            a.heads[2 * bh] = S;
            a.heads[2 * bh + 1] = p.first;
        }
    } else if (a.S == 1) {
        // the last tiles, which see the most keys, of all heads first, and a CU's second workgroup of the short
        // ones, the longer its first is (from an empty cache, 20 heads over 5, 512 / 640 / 1024 / 1400 tokens; the
        // kernel as it was then: 20.9 / 25.4 / 39.7 / 63.4 us; the second in the same order 23.1 / 23.7 / 39.6 /
        // 62.9; head by head from the first tile on 22.4 / 30.5 / 47.6 / 78.6)
        const int w = (int)blockIdx.x, w0 = w >> 8 == 1 && (int)gridDim.x >= 512 ? w ^ 255 : w;
        split = slot = 0;
        S = 1;
        tile = a.tiles - 1 - w0 / a.bh;
        bh = w0 % a.bh;
    } else {
        const int w0 = xcd_order((int)blockIdx.x, (int)gridDim.x), unit = w0 / a.S;
        split = w0 % a.S;
        S = a.S;
        tile = unit % a.tiles;
        bh = unit / a.tiles;
        slot = w0;
    }
    const int b = bh / a.Hkv, kh = bh % a.Hkv, G = a.H / a.Hkv, rows = a.M * G;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    v4f o[NT];
    float top, lrow;
    kv4_rows<HD, RT, STEP, false>(a, bh, tile, split * NW + wave, NW * S, &om[wave][0][0], lane, o, top, lrow);
#pragma unroll
    for (int n = 0; n < NT; ++n) *reinterpret_cast<v4f*>(&om[wave][i][n * 16 + 4 * h]) = o[n];
    if (h == 0) {
        ml[wave][i][0] = top;  // (of a column that saw blocks but none of their keys: -inf, as of one that saw none)
        ml[wave][i][1] = lrow;
    }
    __syncthreads();
    // join the waves' NA columns of a row: 64 NW / RT threads a row
    constexpr int TPR = 64 * NW / RT, NP = NW * NA;
    const int row = t / TPR, RR = tile * RT + row;
    if (RR >= rows) return;
    float mm = -INFINITY, den = 0.0f, f[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) mm = fmaxf(mm, ml[p / NA][p % NA * RT + row][0]);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const float l = ml[p / NA][p % NA * RT + row][1];
        f[p] = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml[p / NA][p % NA * RT + row][0] - mm);
        den += f[p] * l;
    }
    float* dst;
    float inv = 1.0f;
    if (S > 1) {
        float* part = a.work + (size_t)slot * (RT * (HD + 2));
        dst = part + row * HD;
        if (t % TPR == 0) {
            part[RT * HD + 2 * row] = mm;
            part[RT * HD + 2 * row + 1] = den;
        }
    } else {
        dst = a.out + (((size_t)b * a.M + RR / G) * a.H + (size_t)kh * G + RR % G) * HD;
        inv = den;
    }
    constexpr int W = HD / TPR < 4 ? (HD / TPR < 1 ? 1 : HD / TPR) : 4;  // values a thread writes at once
#pragma unroll
    for (int d = t % TPR * W; d < HD; d += TPR * W) {
        float x[W] = {};
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int c = 0; c < W; ++c) x[c] = fmaf(f[p], om[p / NA][p % NA * RT + row][d + c], x[c]);  // (no weight: 0 * 0)
#pragma unroll
        for (int c = 0; c < W; ++c) dst[d + c] = den == 0.0f ? 0.0f : x[c] / inv;
    }
}

// ---- many rows -----------------------------------------------------------------------------
// A workgroup takes a tile of 256 rows (R = m G + g) of one KV head, 32 for each of its 8 waves, over
// blocks of 64 keys.  Together the waves turn a block's codes into keys and values once, as two fp16
// terms each (k 2^a = z 2^a + h 2^a u, the largest of the block in [2^14, 2^15); values with the
// largest so far), into LDS (64 KiB a block at 128 dimensions, two blocks) in the order of the matrix
// instructions; each wave then does, on 32x32x16 products with fp32 sums,
//   S^T = K Q^T and O^T += V^T P^T, each as hi hi + hi lo + lo hi (what is left out is below 2^-22),
// with an online softmax (base 2) per row, rows on lanes: a lane half holds keys 8 (r / 4) +
// 4 (l / 32) + r % 4 of its row in register r, which is the value product's operand as it is.
// The conversion of the next block goes out in pieces of some 12 vector instructions, one under every
// three products of the second half block.  LDS operands are requested two steps (six products)
// before their use, the codes of the block after next while this one is worked on.
// The other way round, codes as exact operands and the scales on the scores as for few rows, does
// with two products of three but asks the vector units for 18 operations a score instead of 9.
// A NaN among the values (a group that reads as NaN) becomes 0 in LDS and is put into the sums of
// the rows that see it afterwards: in a product it would reach every row.
// A key's fp16 terms end at 2^-39 of the block's largest key, a value's at 2^-39 of the largest value so far, a weight's
// at 2^-39 of 1.  That is below fp32's roundings where these (15 h + |z| of their groups, keys of 0 aside) lie within
// 2^11 of each other, and the halves of a row's queries within 2^7.  A split whose keys or values do not, or are below
// 2^-97, whether its rows see them or not, goes through the form for few rows, two tiles of 16 a wave, which scales by
// what a column sees (2048 of 8192 tokens 603 us instead of 400).
// The largest of a wave's upper and lower halves (unsigned, each for itself), in an SGPR.
__device__ __forceinline__ unsigned kv4_wave_max2(unsigned x) {
    typedef unsigned short v2s __attribute__((ext_vector_type(2)));
    auto most = [](unsigned a, unsigned b) {
        return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(v2s, a), __builtin_bit_cast(v2s, b)));
    };
    x = most(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xF, 0xF, false));  // row_ror 1, 2, 4, 8
    x = most(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xF, 0xF, false));
    x = most(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xF, 0xF, false));
    x = most(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xF, 0xF, false));
    const v2u y = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = most(y[0], y[1]);
    const v2u w = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __builtin_amdgcn_readfirstlane(most(w[0], w[1]));
}

constexpr int kKv4Tile = 256;

// A tile of 256 rows in the form for few rows: two tiles of 16 a wave, over the same blocks.
template <int HD>
__device__ __forceinline__ void kv4_far_tile(Kv4AttnArgs a, int w0, int wave, int lane, float* scales) {
    // (what follows from these is worked out here again, and not held through the loop for tiles whose numbers lie near)
    asm("" : "+s"(a.H), "+s"(a.Hkv), "+s"(a.M), "+s"(w0), "+s"(wave), "+v"(lane));
    const int split = w0 % a.S, unit = w0 / a.S, bh = unit % a.bh, tile = a.tiles - 1 - unit / a.bh;
    const int G = a.H / a.Hkv, rows = a.M * G, i = lane & 15;
    float* const part = a.work + ((size_t)((size_t)bh * a.tiles + tile) * a.S + split) * (kKv4Tile * (HD + 2));
#pragma unroll 1
    for (int sub = 2 * wave; sub < 2 * wave + 2; ++sub) {
        const int tile16 = tile * (kKv4Tile / 16) + sub, R = tile16 * 16 + i;
        if (tile16 * 16 >= rows) break;
        v4f x[HD / 16];
        float top, sum;
        kv4_rows<HD, 16, false, true>(a, bh, tile16, split, a.S, scales, lane, x, top, sum);
        if (R >= rows) continue;
        float* dst = part + (sub * 16 + i) * HD;
        float over = 1.0f;
        if (a.S > 1) {
            part[kKv4Tile * HD + 2 * (sub * 16 + i)] = top;
            part[kKv4Tile * HD + 2 * (sub * 16 + i) + 1] = sum;
        } else {
            dst = a.out + (((size_t)(bh / a.Hkv) * a.M + R / G) * a.H + (size_t)(bh % a.Hkv) * G + R % G) * HD;
            over = sum;
        }
#pragma unroll
        for (int n = 0; n < HD / 16; ++n) {
#pragma unroll
            for (int r = 0; r < 4; ++r) x[n][r] = sum == 0.0f ? 0.0f : x[n][r] / over;
            *reinterpret_cast<v4f*>(dst + 16 * n + (lane >> 4) * 4) = x[n];
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(512, 2) kv4_prefill_kernel(const Kv4AttnArgs a) {
    constexpr int NG = HD / 64, NU = HD / 32, OCT = HD / 8, TR = kKv4Tile;
    constexpr int PLANE = OCT * 64, BUF = 4 * PLANE;  // 16-byte units: K hi, K lo, V hi, V lo
    __shared__ v2u span[8];  // of every eighth block, one wave's: `near`
    extern __shared__ __attribute__((aligned(16))) v8h lds_kv4[];  // two blocks of
    // keys [octet of dimensions][64] and values [4 w + 2 s + l][HD], hi then lo
    // the last tiles see the most keys: they go out first, of all heads
    const int w0 = (int)blockIdx.x, split = w0 % a.S, unit0 = w0 / a.S, bh = unit0 % a.bh, tile = a.tiles - 1 - unit0 / a.bh;
    const int b = bh / a.Hkv, kh = bh % a.Hkv, G = a.H / a.Hkv;
    const int t = threadIdx.x, lane = t & 63, c32 = lane & 31, hl = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const unsigned mask = kv4_mask();
    const int pos = a.pos[b];
    const int rows = a.M * G, R0 = tile * TR + wave * 32, R = min(R0 + c32, rows - 1), m = R / G;
    const int last = kv4_row_pos(pos, m, a.Lmax);
    const int kend = kv4_range(pos, tile * TR / G, (min(tile * TR + TR, rows) - 1) / G, a.Lmax).kend;
    // what the wave's rows see
    const Kv4Range mine = kv4_range(pos, min(R0, rows - 1) / G, (min(R0 + 32, rows) - 1) / G, a.Lmax);
    const int lo_last = mine.all, hi_last = R0 < rows ? mine.kend - 1 : -1;
    const int nb = (kend + kKv4Block - 1) / kKv4Block;
    const uint8_t* const head = a.cache + (size_t)bh * a.nblk * kv4_block_bytes(HD);
    // This thread's part of a block.  Keys: of key `lane`, lane group ch = wave % 4, group wave / 4 (64
    // dimensions: octet wave / 4).  Values: dimensions (u, v, d), (u, d) = vl, over the keys of lane group ch
    // of half wv (64 dimensions: v = wave / 4), with these keys' scales.  And the scales of key `lane`, from
    // which every wave finds the block's largest numbers.
    const int ch = wave & 3, cg = wave >> 2;
    const int vl = HD == 128 ? lane : lane & 31, wv = HD == 128 ? cg : lane >> 5;
    const int vkey = 32 * wv + 16 * (ch >> 1) + 4 * (ch & 1);  // first of its keys: + (0..3, 8..11)
    // (byte offsets in a block, whose address is uniform)
    const unsigned at_k = (lane * OCT + ch * 2 * NG + cg * NG) * 4,
                   at_v = 32 * HD + ((vl * 4 + ch) * 4 + wv + (NG == 2 ? 0 : 2 * cg)) * 4,
                   at_s = 64 * HD + lane * 4, at_vs = 68 * HD + ((vl >> 5) * 64 + vkey) * 4;
    unsigned kc[NG], vc[NG], ks[NG], vk[NG];
    v4u vs[2];
    const uint8_t* blk = head;  // the block that is loaded
    auto word = [&](unsigned at) __attribute__((always_inline)) { return *reinterpret_cast<const unsigned*>(blk + at); };
    constexpr int LK = 2 * NG, LV = 2 * NG + 2;  // loads of the keys' and of the values' part
    auto load_k = [&](int n) __attribute__((always_inline)) {
        if (n < NG) kc[n] = word(at_k + 4 * n);
        else ks[n - NG] = word(at_s + 256 * (n - NG));
    };
    auto load_v = [&](int n) __attribute__((always_inline)) {
        if (n < NG) vc[n] = word(at_v + 8 * n);
        else if (n < 2 * NG) vk[n - NG] = word(at_s + 4 * HD + 256 * (n - NG));
        else vs[n - 2 * NG] = *reinterpret_cast<const v4u*>(blk + (at_vs + 32 * (n - 2 * NG)));
    };
    auto load_ks = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < LK; ++n) load_k(n);
    };
    auto load_vs = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < LV; ++n) load_v(n);
    };
    // the block's codes -> LDS; what the products over it need to know
    struct Blk {
        float c;    // scores' factor but for the row's
        float fix;  // factor of the sums so far
        unsigned long long nan[NG];  // keys whose values read as NaN, by group
    };
    int ve = -111;  // exponent of the largest value so far
    float kf = 0.0f, vf = 0.0f;
    // the block in registers, before its conversion: `more` false: there is none
    auto prepare = [&](int j, bool more) __attribute__((always_inline)) {
        const int key0 = j * kKv4Block;
        Blk n;
        if (key0 + kKv4Block > kend) {  // what lies behind the newest key is not read as a number
#pragma unroll
            for (int g = 0; g < NG; ++g)
                if (key0 + lane >= kend) ks[g] = vk[g] = 0u;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (key0 + vkey + 8 * x + r >= kend) vs[x][r] = 0u;
        }
        float kmax = 0.0f, vmax = 0.0f;
        unsigned long long nans = 0ull;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            kmax = fmaxf(kmax, fmaf(15.0f, kv4_h(ks[g]), fabsf(kv4_z(ks[g]))));
            vmax = fmaxf(vmax, fmaf(15.0f, kv4_h(vk[g]), fabsf(kv4_z(vk[g]))));
            n.nan[g] = __ballot((vk[g] & 0x7F800000u) == 0x7F800000u);
            nans |= n.nan[g];
        }
        if (nans != 0ull)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if ((vs[x][r] & 0x7F800000u) == 0x7F800000u) vs[x][r] = 0u;
        // (their exponents' order is that of their upper halves)
        const unsigned top2 = kv4_wave_max2(__float_as_uint(kmax) >> 16 | (__float_as_uint(vmax) & 0xFFFF0000u));
        const int ke = min(max((int)(top2 >> 7 & 255u) - 127, -111), 127);
        const int vn = more ? min(max((int)(top2 >> 23) - 127, ve), 127) : ve;
        kf = kv4_pow2(14 - ke);
        vf = kv4_pow2(14 - vn);
        n.c = kv4_pow2(ke - 14);
        n.fix = ve - vn < -126 ? 0.0f : kv4_pow2(ve - vn);
        ve = vn;
        return n;
    };
    // piece k of its conversion: elements 2 (k % 4), .. + 1 of dword k / 4, and a dword's stores with its last
    v4u chi, clo;
    auto piece = [&](unsigned w, int k, float z0, float h0, float z1, float h1, v8h* hi_at, v8h* lo_at)
                     __attribute__((always_inline)) {
        const v2h u = kv4_level2(w, k % 4, mask);
        v2h hi, lo;
        kv4_split(v2f{fmaf((float)u[0], h0, z0), fmaf((float)u[1], h1, z1)}, hi, lo);
        chi[k % 4] = __builtin_bit_cast(unsigned, hi);
        clo[k % 4] = __builtin_bit_cast(unsigned, lo);
        if (k % 4 == 3) {
            *hi_at = __builtin_bit_cast(v8h, chi);
            *lo_at = __builtin_bit_cast(v8h, clo);
        }
    };
    auto piece_k = [&](int k, v8h* buf) __attribute__((always_inline)) {
        // 128 dimensions: octets 8 g + 2 ch + e; 64: octet 2 ch + wave / 4
        const unsigned own = NG == 2 && cg ? ks[NG - 1] : ks[0];
        const float z = kv4_z(own) * kf, h = kv4_h(own) * kf;
        v8h* const at = buf + (NG == 2 ? 8 * cg + 2 * ch + k / 4 : 2 * ch + cg) * 64 + lane;
        piece(kc[k / 4], k, z, h, z, h, at, at + PLANE);
    };
    auto piece_v = [&](int k, v8h* buf) __attribute__((always_inline)) {
        const unsigned s0 = vs[k % 4 / 2][k % 2 * 2], s1 = vs[k % 4 / 2][k % 2 * 2 + 1];
        v8h* const at = buf + 2 * PLANE + (4 * wv + ch) * HD + vl / 16 * 32 + 16 * (NG == 2 ? k / 4 : cg) + vl % 16;
        piece(vc[k / 4], k, kv4_z(s0) * vf, kv4_h(s0) * vf, kv4_z(s1) * vf, kv4_h(s1) * vf, at, at + PLANE);
    };
    auto convert = [&](v8h* buf) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 4 * NG; ++k) piece_k(k, buf);
#pragma unroll
        for (int k = 0; k < 4 * NG; ++k) piece_v(k, buf);
    };
    if (split < nb) {
        blk = head + (size_t)split * kv4_block_bytes(HD);
        load_ks();
        load_vs();
    }
    // The largest 15 h + |z| of the keys (lower half) and values (upper half) of every eighth block, and the smallest's
    // complement (keys of 0 aside), the upper halves of the fp32 bits.  (In the loop, block by block, the same took 2 %
    // of the launch, however it was spread.)
    float kmax = 0.0f, kmin = INFINITY, vmax = 0.0f, vmin = INFINITY;
    for (int j0 = split + wave * a.S; j0 < nb; j0 += 32 * a.S) {
        unsigned sc[4][2 * NG];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int g = 0; g < 2 * NG; ++g)
                sc[c][g] = *reinterpret_cast<const unsigned*>(head + (size_t)min(j0 + 8 * c * a.S, nb - 1) * kv4_block_bytes(HD) + (at_s + 256 * g));
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const bool in = min(j0 + 8 * c * a.S, nb - 1) * kKv4Block + lane < kend;
#pragma unroll
            for (int g = 0; g < 2 * NG; ++g) {
                const float x = in ? fmaf(15.0f, kv4_h(sc[c][g]), fabsf(kv4_z(sc[c][g]))) : __builtin_nanf("");
                if (g < NG) {
                    kmax = fmaxf(kmax, x);
                    kmin = x == 0.0f ? kmin : fminf(kmin, x);
                } else {
                    vmax = fmaxf(vmax, x);
                    vmin = fminf(vmin, x);
                }
            }
        }
    }
    v2u near = {kv4_wave_max2(__float_as_uint(kmax) >> 16 | (__float_as_uint(vmax) & 0xFFFF0000u)),
                      kv4_wave_max2(~(__float_as_uint(kmin) >> 16 | (__float_as_uint(vmin) & 0xFFFF0000u)))};
    // A wave's rows pass through its part of LDS, queries here and results at the end, so that memory is read
    // and written in whole lines (lane by lane, 32 rows at once, the launch took some 1000 cycles more): 16-byte unit c
    // of row r lies at unit c ^ (r % 16).  Coalesced, instruction n takes rows n RPI + lane / UPR, unit lane % UPR.
    constexpr int UPR = HD / 4, RPI = 64 / UPR;
    v4f* const own = reinterpret_cast<v4f*>(lds_kv4) + wave * 32 * UPR;
    auto in_lds = [&](int r, int c) __attribute__((always_inline)) { return own + r * UPR + (c ^ (r & 15)); };
    const int mw = R0 / G;
    const float inv_g = 1.0f / (float)G;
    auto row_at = [&](int r) __attribute__((always_inline)) {  // (row R0 + r of this KV head) * HD
        const int x = min(R0 + r, rows - 1) - mw * G, dm = (int)(((float)x + 0.5f) * inv_g);
        return (((size_t)b * a.M + mw + dm) * a.H + (size_t)kh * G + (x - dm * G)) * HD;
    };
    // the row's queries: dimensions 16 s + 8 hl + (0..7) in lane half hl
    float qi;
    v8h qh[OCT / 2], ql[OCT / 2];
    {
        if (R0 < rows)
#pragma unroll
            for (int n = 0; n < 32 / RPI; ++n) {
                const int r = n * RPI + lane / UPR;
                *in_lds(r, lane % UPR) = *reinterpret_cast<const v4f*>(a.q + row_at(r) + lane % UPR * 4);
            }
        kv4_wave_lds();
        float qx[OCT / 2][8], big[NG] = {};
#pragma unroll
        for (int s = 0; s < OCT / 2; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const v4f x = *in_lds(c32, 4 * s + 2 * hl + e);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    qx[s][4 * e + c] = x[c] * a.scale;
                    big[s / 4] = fmaxf(big[s / 4], fabsf(qx[s][4 * e + c]));
                }
            }
#pragma unroll
        for (int g = 0; g < NG; ++g) big[g] = kv4_join32(big[g], Kv4Max());
        const int qe = kv4_query_power(fmaxf(big[0], big[NG - 1]));
        if constexpr (NG == 2)  // (a half that is far smaller: kv4_far_tile)
            if (R0 < rows && __any(fminf(big[0], big[1]) > 0.0f && fmaxf(big[0], big[1]) < INFINITY && abs(kv4_exponent(big[0]) - kv4_exponent(big[1])) > 6)) near[0] |= 0x8000u;
        const float qf = kv4_pow2(qe);
        qi = kv4_pow2(-qe);
#pragma unroll
        for (int s = 0; s < OCT / 2; ++s)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                v2h hi, lo;
                kv4_split(v2f{qx[s][e] * qf, qx[s][e + 1] * qf}, hi, lo);
                qh[s][e] = hi[0];
                qh[s][e + 1] = hi[1];
                ql[s][e] = lo[0];
                ql[s][e + 1] = lo[1];
            }
    }
    v16f o[NU];
    float top = -INFINITY, off = 14.0f, lrow = 0.0f;
#pragma unroll
    for (int u = 0; u < NU; ++u) o[u] = v16f{};
    Blk cur{}, next{};
    // 32 keys (half w of a block): scores, softmax, values.  With NEXT, a piece of the next block's
    // conversion goes out under every three products.
    auto multiply = [&](auto w_, auto next_, int j, const v8h* buf, v8h* other) __attribute__((always_inline)) {
        constexpr int w = decltype(w_)::value;
        constexpr bool NEXT = decltype(next_)::value;
        const int key0 = j * kKv4Block + 32 * w;
        const v8h* const lk = buf + 32 * w + c32 + hl * 64;
        const v8h* const lv = buf + 2 * PLANE + (4 * w + hl) * HD + c32;
        constexpr int QS = OCT / 2, VS = 2 * NU, AHEAD = 2;
        v8h rh[AHEAD + 1], rl[AHEAD + 1];
        auto fetch = [&](int k) __attribute__((always_inline)) {  // operands of step k: QS of the scores, then VS of the values
            if (k < QS) {
                rh[k % (AHEAD + 1)] = lk[2 * k * 64];
                rl[k % (AHEAD + 1)] = lk[PLANE + 2 * k * 64];
            } else if (k < QS + VS) {
                const int u = (k - QS) / 2, x = (k - QS) % 2;
                rh[k % (AHEAD + 1)] = lv[2 * x * HD + 32 * u];
                rl[k % (AHEAD + 1)] = lv[PLANE + 2 * x * HD + 32 * u];
            }
        };
        auto spread = [&]() __attribute__((always_inline)) {  // a step's instructions: products, vector work between them
            if constexpr (NEXT) {
#pragma unroll
                for (int n = 0; n < 3; ++n) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) fetch(k);
        v16f s = v16f{};
#pragma unroll
        for (int k = 0; k < QS; ++k) {
            fetch(k + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(rh[k % (AHEAD + 1)], qh[k], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(rh[k % (AHEAD + 1)], ql[k], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(rl[k % (AHEAD + 1)], qh[k], s, 0, 0, 0);
            if constexpr (NEXT) piece_k(k, other);
            else if (k >= QS - LV) load_v(k - (QS - LV));  // (a load holds the wave some 60 cycles: under the products)
            spread();
        }
        // (queries of 0 over small keys: the product of the factors falls to 0, and -inf times 0 is NaN)
        const float c = fmaxf(qi * cur.c, 0x1p-126f), fix = w == 0 ? cur.fix : 1.0f;
        if (key0 + 31 > lo_last)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = key0 + 8 * (r >> 2) + 4 * hl + (r & 3) <= last ? s[r] : -INFINITY;
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        const float now = fmaxf(top, kv4_join32(mx, Kv4Max()) * c);
        if (__any(now != top) || fix != 1.0f) {
            // weights are 2^(s + off), up to 2^14 (beside a score of 2^25 and more the 14 may round to 16, an
            // infinity in fp16)
            const float ref = now == -INFINITY ? 0.0f : now, old = off;
            off = (14.0f - ref) + ref < 15.0f ? 14.0f - ref : -ref;
            const float alpha = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(off - old);
            lrow *= alpha;
#pragma unroll
            for (int u = 0; u < NU; ++u) o[u] *= alpha * fix;
            top = now;
        }
        v8h ph[2], pl[2];
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
            float p0 = __builtin_amdgcn_exp2f(fmaf(s[r], c, off)), p1 = __builtin_amdgcn_exp2f(fmaf(s[r + 1], c, off));
            v2h hi, lo;
            kv4_split(p0, p1, hi, lo);
            lrow += p0 + p1;
            ph[r >> 3][r & 7] = hi[0];
            ph[r >> 3][(r & 7) + 1] = hi[1];
            pl[r >> 3][r & 7] = lo[0];
            pl[r >> 3][(r & 7) + 1] = lo[1];
        }
#pragma unroll
        for (int k = QS; k < QS + VS; ++k) {
            fetch(k + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
            const int u = (k - QS) / 2, x = (k - QS) % 2;
            o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(rh[k % (AHEAD + 1)], ph[x], o[u], 0, 0, 0);
            o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(rh[k % (AHEAD + 1)], pl[x], o[u], 0, 0, 0);
            o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(rl[k % (AHEAD + 1)], ph[x], o[u], 0, 0, 0);
            if constexpr (NEXT) piece_v(k - QS, other);
            if (NEXT && k >= QS + VS - LK) load_k(k - (QS + VS - LK));
            spread();
        }
    };
    using Half0 = std::integral_constant<int, 0>;
    using Half1 = std::integral_constant<int, 1>;
    // The registers hold the keys' part of block j + S when block j is begun; its values' part follows.
    // Behind the last block the last one is loaded, and converted into a buffer that is not read.
    auto block_at = [&](int j) __attribute__((always_inline)) { return head + (size_t)min(j, nb - 1) * kv4_block_bytes(HD); };
    if (lane == 0) span[wave] = near;
    __syncthreads();  // (the waves' parts for the queries are the first block's)
    {
        const v2u x = span[lane & 7];
        const unsigned hi = kv4_wave_max2(x[0]), lo = ~kv4_wave_max2(x[1]);  // exponents of keys: bits 7.., of values: bits 23..
        const int kn = hi >> 7 & 255u, kl = lo >> 7 & 255u, vn = hi >> 23 & 255u, vl = lo >> 23 & 255u;
        if (__builtin_expect((hi & 0x8000u) != 0u || kl < max(kn - 10, 30) || (vn != 0 && vl < max(vn - 10, 30)), 0)) {
            kv4_far_tile<HD>(a, (int)blockIdx.x, wave, lane, reinterpret_cast<float*>(own));
            return;
        }
    }
    if (split < nb) {
        cur = prepare(split, true);
        convert(lds_kv4);
        blk = block_at(split + a.S);
        load_ks();
    }
    __syncthreads();
    int side = 0;
    for (int j = split; j < nb; j += a.S, side ^= 1) {
        v8h *const buf = lds_kv4 + side * BUF, *const other = lds_kv4 + (side ^ 1) * BUF;
        const bool more = j + a.S < nb;
        blk = block_at(j + a.S);
        if (j * kKv4Block <= hi_last || cur.fix != 1.0f) {
            // of a SIMD's two waves one goes first in the first half, the other in the second
            if (wave < 4) __builtin_amdgcn_s_setprio(1);
            multiply(Half0{}, std::false_type{}, j, buf, other);
            if (wave < 4) __builtin_amdgcn_s_setprio(0);
            else __builtin_amdgcn_s_setprio(1);
            next = prepare(j + a.S, more);
            blk = block_at(j + 2 * a.S);
            multiply(Half1{}, std::true_type{}, j, buf, other);
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int g = 0; g < NG; ++g)
                for (unsigned long long nans = cur.nan[g]; nans != 0ull; nans &= nans - 1) {  // (rare)
                    const bool see = j * kKv4Block + (int)__builtin_ctzll(nans) <= last;
#pragma unroll
                    for (int u = 2 * g; u < 2 * g + 2; ++u)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[u][r] = see ? __builtin_nanf("") : o[u][r];
                }
        } else {  // none of the wave's rows sees the block
            load_vs();
            next = prepare(j + a.S, more);
            convert(other);
            blk = block_at(j + 2 * a.S);
            load_ks();
        }
        __syncthreads();
        cur = next;
    }
    // O[row][dim]: dimensions 32 u + 8 (r / 4) + 4 hl + r % 4 of the lane's row
    lrow = kv4_join32(lrow, Kv4Sum());
    if (R0 >= rows) return;
    const float back = kv4_pow2(max(ve - 14, -126)), inv = a.S > 1 ? 1.0f : lrow == 0.0f ? 0.0f : 1.0f / lrow;
    float* const part = a.work + ((size_t)((size_t)bh * a.tiles + tile) * a.S + split) * (TR * (HD + 2));
    if (a.S > 1 && hl == 0) {
        part[TR * HD + 2 * (wave * 32 + c32)] = lrow == 0.0f ? -INFINITY : -off;
        part[TR * HD + 2 * (wave * 32 + c32) + 1] = lrow;
    }
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            v4f x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = o[u][r + e] * inv * back;
            *in_lds(c32, 8 * u + r / 2 + hl) = x;
        }
    kv4_wave_lds();
#pragma unroll
    for (int n = 0; n < 32 / RPI; ++n) {
        const int r = n * RPI + lane / UPR;
        float* const dst = a.S > 1 ? part + (wave * 32 + r) * HD : a.out + row_at(r);
        const v4f x = *in_lds(r, lane % UPR);
        if (R0 + r < rows) *reinterpret_cast<v4f*>(dst + lane % UPR * 4) = x;
    }
}

// out from the S partials of every unit (tiles of TR rows).  A row takes HD / 4 lanes, four values
// each, in sg copies that share its splits: 1 where there are rows enough to fill the GPU, else all
// of the workgroup's (1024 threads where there are many splits, so that each lane has few loads, all
// in flight at once).
template <int HD>
__global__ void __launch_bounds__(1024) kv4_combine_kernel(const Kv4AttnArgs a, int TR, int sg) {
    constexpr int LR = HD / 4, AT = 4;
    __shared__ v4f sx[16 * LR];
    __shared__ float sd[16];
    const int t = threadIdx.x, c = t % LR, grp = t / LR;
    const int G = a.H / a.Hkv, rows = a.M * G, most = min(TR, rows);  // (a tile's rows that can be live)
    const long long rr = (long long)blockIdx.x * ((int)blockDim.x / LR / sg) + grp / sg;  // (unit, row of the tile)
    const long long unit = rr / most;
    const int row = (int)(rr % most), tile = (int)(unit % a.tiles), bh = (int)(unit / a.tiles), R = tile * TR + row;
    const bool live = unit < (long long)a.bh * a.tiles && R < rows;
    const size_t psz = (size_t)TR * (HD + 2);
    int S = a.S;
    size_t slot = (size_t)unit * S;
    if (S == 0) {
        S = a.heads[live ? 2 * bh : 0];
        slot = (size_t)a.heads[live ? 2 * bh + 1 : 1];
    }
    const float* part = a.work + (live ? slot : 0) * psz;
    const float *pm = part + (size_t)TR * HD + 2 * (live ? row : 0), *po = part + (size_t)(live ? row : 0) * HD + 4 * c;
    float mm = -INFINITY;
    for (int s = c; s < S; s += LR) mm = fmaxf(mm, pm[s * psz]);
    v4f x{};
    float den = 0.0f;
    bool first = true;
    for (int s0 = grp % sg; s0 < S || first; s0 += AT * sg) {
        v4f y[AT];
        float m[AT], l[AT];
#pragma unroll
        for (int k = 0; k < AT; ++k) {
            const int s = s0 + k * sg;
            const bool in = s < S;
            m[k] = in ? pm[s * psz] : 0.0f;
            l[k] = in ? pm[s * psz + 1] : 0.0f;
            y[k] = in ? *reinterpret_cast<const v4f*>(po + s * psz) : v4f{};
        }
        if (first) {  // (the first loads are on their way meanwhile)
#pragma unroll
            for (int w = 1; w < LR; w <<= 1) mm = fmaxf(mm, __shfl_xor(mm, w, 64));
            first = false;
        }
#pragma unroll
        for (int k = 0; k < AT; ++k) {
            const float f = l[k] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m[k] - mm);
            den = fmaf(f, l[k], den);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = fmaf(f, y[k][e], x[e]);  // (no weight: 0 * 0)
        }
    }
    if (sg > 1) {  // (one row a workgroup: lanes c, c + LR, .. of every wave, then the waves)
#pragma unroll
        for (int w = LR; w < 64; w <<= 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], w, 64);
            den += __shfl_xor(den, w, 64);
        }
        const int waves = (int)blockDim.x / 64;
        if ((t & 63) < LR) {
            sx[t / 64 * LR + c] = x;
            if (c == 0) sd[t / 64] = den;
        }
        __syncthreads();
        if (t >= LR) return;
        for (int k = 1; k < waves; ++k) {
            x += sx[k * LR + c];
            den += sd[k];
        }
    }
    if (!live || S == 1) return;  // (in one piece: written already)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = den == 0.0f ? 0.0f : x[e] / den;
    *reinterpret_cast<v4f*>(a.out + (((size_t)(bh / a.Hkv) * a.M + R / G) * a.H + (size_t)(bh % a.Hkv) * G + R % G) * HD +
                            4 * c) = x;
}

// Workgroups of 256 in one launch: its work items are counted in 32 bits.
constexpr long long kMaxGroups = 0xFFFFFFFFll / 256;

hipError_t kv4_prepare_device() {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(&kv4_prefill_kernel<128>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, 1024 * 128);
}

size_t kv4_bytes(int B, int Hkv, int hd, int Lmax) {
    return (size_t)B * Hkv * ((Lmax + kKv4Block - 1) / kKv4Block) * kv4_block_bytes(hd);
}

hipError_t launch_kv4_append(const float* q, const float* k, const float* v, const float* rope, void* cache,
                             float* q_out, int B, int M, int H, int Hkv, int hd, int Lmax, const int* pos,
                             hipStream_t s) {
    const int nblk = (Lmax + kKv4Block - 1) / kKv4Block, chunks = (M + kKv4Rows - 2) / kKv4Rows + 1;
    const long long nkv = (long long)B * Hkv * chunks, nq = ((long long)B * M * H * (hd / 8) + 255) / 256;
    if (nkv + nq > kMaxGroups) return hipErrorInvalidValue;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(nkv + nq)), dim3(256), 0, s, q, k, v, rope,
                           static_cast<uint8_t*>(cache), q_out, B, M, H, Hkv, Lmax, nblk, chunks, (int)nkv, pos);
    };
    if (hd == 128) go(kv4_append_kernel<128>);
    else go(kv4_append_kernel<64>);
    return hipGetLastError();
}

hipError_t launch_kv4_read(const void* cache, float* k, float* v, int B, int M, int Hkv, int hd, int Lmax,
                           const int* pos, hipStream_t s) {
    const int nblk = (Lmax + kKv4Block - 1) / kKv4Block;
    const int chunks = (M + kKv4Block - 2) / kKv4Block + 1;
    const long long n = (long long)B * Hkv * chunks;
    if (n > kMaxGroups) return hipErrorInvalidValue;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(256), 0, s, static_cast<const uint8_t*>(cache), k, v, M, Hkv,
                           Lmax, nblk, chunks, pos);
    };
    if (hd == 128) go(kv4_read_kernel<128>);
    else go(kv4_read_kernel<64>);
    return hipGetLastError();
}

namespace {
// Which kernel, and how many splits of the keys.  The host does not know the positions: the tile is chosen
// as for a call at its cache's end, the splits as half way into it.  (Times: 20 heads of 128 over 5, the
// launches back to back.)
struct Kv4Shape {
    long long units, groups;  // groups: workgroups of the attention launch, and partials
    int RT, tiles, S;         // S = 0: by length (kv4_piece)
    int NW;                   // waves a workgroup (tiles of up to 16 rows)
};
Kv4Shape kv4_shape(int B, int M, int H, int Hkv, int hd, int Lmax) {
    Kv4Shape p;
    const long long rows = (long long)M * (H / Hkv), t16 = (rows + 15) / 16, big = (rows + kKv4Tile - 1) / kKv4Tile;
    const int blocks = (Lmax + kKv4Block - 1) / kKv4Block;
    // 256 rows in one tile or in 16 of 16 rows.  A big tile's launch costs more before it pays (its queries and
    // results pass through one workgroup a CU) and its conversion of every block however few its rows, a small
    // one each block's codes again.  Per block of 64 keys at 128 dimensions, a big tile takes 9.3 ns and 0.75 for
    // every 16 rows in it, a small one 1.8; at 64, 6.5 and 0.32 against 0.82.  In tiles of 16 / 256 rows, us, 20
    // heads over 5: 16 sequences of 24 tokens at 4000 71 / 102, of 48 128 / 130, of 64 152 / 145, 4 of 64 61 / 53,
    // of 96 63 / 88; 1400 tokens from an empty cache 54 / 69, 2000 92 / 93, 512 after 1500 48 / 52, after 2500
    // 68 / 61, 128 after 8192 53 / 56, 192 75 / 66; 32 heads over 8, 700 after 700 57 / 67, 300 after 4000 95 / 105,
    // 1000 after 1000 100 / 102; 16 heads of 64 over 8, 2000 after 2000 90 / 98, 2048 after 6144 198 / 195, two of
    // those 383 / 362.
    const double gain = (hd == 128 ? 1.05 * t16 - 9.3 * big : 0.5 * t16 - 6.5 * big) * B * Hkv * (Lmax - M / 2) / kKv4Block;
    p.RT = rows <= 4 ? 4 : rows <= 8 ? 8 : gain < (hd == 128 ? 11500.0 : 18000.0) ? 16 : kKv4Tile;
    const long long tiles = (rows + p.RT - 1) / p.RT;
    p.tiles = (int)std::min(tiles, 0x7FFFFFFFll);
    p.units = (long long)B * Hkv * tiles;
    // A split's results pass through memory and a second launch (3 to 16 us), so there is none where a
    // wave has 5 blocks or fewer without (8 sequences of 12 heads over 777 keys 7.9 us, in 4 splits 9.6), and
    // a tile of 256 rows keeps 8 blocks a split (128 tokens after 8192: 16 splits 57 us, 24 62).  Else as many
    // as two workgroups a CU take in one round, the big tiles, one a CU, in two: one token over 1538 keys
    // in 8 / 4 / 1 splits 10.6 / 12.4 / 17.7 us, over 131072 in 200 / 102 / 50 35.9 / 30.7 / 33.2; 2048 of 8192
    // tokens in 1 / 2 / 3 / 5 splits 507 / 504 / 405 / 476 (in equal runs of blocks over 256 workgroups, a unit
    // cut where a run ends, as long as in 3: the clock gives way to the matrix cores' power).
    const int fours = (blocks + 3) / 4;
    int most = p.RT == kKv4Tile ? blocks / 8 : blocks <= 20 ? 1 : fours, wide = 512;
    // Tiles of 16 rows: a workgroup's keys over eight waves instead of four, one workgroup a CU, but where every
    // wave of four takes one block at most, or two in a short cache.  In four / eight, us: 16 tokens at 620 (100)
    // 12.2 / 10.6 (7.3 / 7.9), at 2400 (3800, 8000) 11.8 / 13.7 (14.5 / 14.0, 20.3 / 17.8), 64 at 2400 19.9 / 18.9,
    // 160 at 1300 (8000) 25.8 / 17.1 (69.6 / 62.2), 3 x 77 at 900 (14 heads of 64 over 2) 9.9 / 9.2.  Four or
    // eight rows a tile, one token at 1279 (639, 450) 13.7 / 13.3 (10.1 / 10.2, 8.4 / 9.3): not there.
    p.NW = 4;
    if (p.RT == 16 && p.units <= 256 && blocks > 8 && (blocks <= 20 || p.units * fours > 256)) {
        p.NW = 8;
        most = blocks <= 20 ? 1 : (blocks + 7) / 8;
        wide = 256;
    }
    p.S = (int)std::max(1ll, std::min<long long>(most, wide / p.units));
    p.groups = p.units * p.S;
    // A batch: splits by length.  Sequences of 100 to 4096 keys, 32 / 8 / 48 of them: 24.0 / 14.3 / 30.3 us,
    // with the best equal number of splits 25.5 / 14.6 / 33.3; 4 of 100 to 32768 22.6 / 28.3; 50 of 100 to 1500
    // (250 heads, few keys) 20.2 / 17.1, so not there; 32 of 4096 each 30.0 / 28.6.
    if (B > 1 && B <= 64 && tiles == 1 && p.RT != kKv4Tile && p.units <= kKv4Slots / 2 &&
        blocks > (p.units <= kKv4Slots / 4 ? 20 : 31)) {
        p.S = 0;
        p.NW = 4;
        p.groups = kKv4Slots;
    }
    return p;
}
template <int HD, bool STEP>
void run_kv4_few(const Kv4AttnArgs& a, const Kv4Shape& p, hipStream_t s) {
    const dim3 grid((unsigned)p.groups), block(64 * p.NW);
    if (p.RT == 4) hipLaunchKernelGGL((kv4_attn_kernel<HD, 4, STEP, 4>), grid, block, 0, s, a);
    else if (p.RT == 8) hipLaunchKernelGGL((kv4_attn_kernel<HD, 8, STEP, 4>), grid, block, 0, s, a);
    else if (p.NW == 4) hipLaunchKernelGGL((kv4_attn_kernel<HD, 16, STEP, 4>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((kv4_attn_kernel<HD, 16, STEP, 8>), grid, block, 0, s, a);
}
template <int HD>
hipError_t run_kv4_attention(const Kv4AttnArgs& a, const Kv4Shape& p, hipStream_t s) {
    if (a.put) run_kv4_few<HD, true>(a, p, s);
    else if (p.RT != kKv4Tile) run_kv4_few<HD, false>(a, p, s);
    else hipLaunchKernelGGL(kv4_prefill_kernel<HD>, dim3((unsigned)p.groups), dim3(512), 1024 * HD, s, a);
    if (p.S != 1) {
        const long long all = p.units * std::min<long long>(p.RT, (long long)a.M * (a.H / a.Hkv));  // rows
        const int threads = (p.S == 0 ? p.groups / p.units : p.S) > 16 && all < 4096 ? 1024 : 256, gr = threads / (HD / 4), sg = all >= 4096 ? 1 : gr;
        hipLaunchKernelGGL(kv4_combine_kernel<HD>, dim3((unsigned)((all * sg + gr - 1) / gr)), dim3(threads), 0, s, a, p.RT,
                           sg);
    }
    return hipGetLastError();
}
}  // namespace

size_t kv4_attention_workspace(int B, int M, int H, int Hkv, int hd, int Lmax) {
    const Kv4Shape p = kv4_shape(B, M, H, Hkv, hd, Lmax);
    return p.S == 1 ? 0 : (size_t)p.groups * p.RT * (hd + 2) * sizeof(float) + (p.S == 0 ? (size_t)p.units * 8 : 0);
}

namespace {
hipError_t launch_kv4(Kv4AttnArgs a, int B, int hd, hipStream_t s) {
    const Kv4Shape p = kv4_shape(B, a.M, a.H, a.Hkv, hd, a.Lmax);
    if (p.groups > (p.RT == kKv4Tile ? kMaxGroups / 2 : kMaxGroups)) return hipErrorInvalidValue;
    a.nblk = (a.Lmax + kKv4Block - 1) / kKv4Block;
    a.tiles = p.tiles;
    a.S = p.S;
    a.bh = B * a.Hkv;
    a.heads = reinterpret_cast<int*>(a.work + (p.S == 0 ? (size_t)p.groups * p.RT * (hd + 2) : 0));
    a.scale = 1.44269504088896341f / sqrtf((float)hd);
    return hd == 128 ? run_kv4_attention<128>(a, p, s) : run_kv4_attention<64>(a, p, s);
}
}  // namespace

hipError_t launch_kv4_attention(const float* q, const void* cache, float* out, int B, int M, int H, int Hkv, int hd,
                                int Lmax, const int* pos, float* work, hipStream_t s) {
    Kv4AttnArgs a{};
    a.q = q;
    a.cache = static_cast<const uint8_t*>(cache);
    a.out = out;
    a.work = work;
    a.pos = pos;
    a.M = M;
    a.H = H;
    a.Hkv = Hkv;
    a.Lmax = Lmax;
    return launch_kv4(a, B, hd, s);
}

// One token a sequence: append and attention (H / Hkv <= 16: a head is one tile, and its new row one wave's).
hipError_t launch_kv4_step(const float* q, const float* k, const float* v, const float* rope, void* cache, float* out,
                           int B, int H, int Hkv, int hd, int Lmax, const int* pos, float* work, hipStream_t s) {
    Kv4AttnArgs a{};
    a.q = q;
    a.cache = a.put = static_cast<uint8_t*>(cache);
    a.out = out;
    a.work = work;
    a.pos = pos;
    a.M = 1;
    a.H = H;
    a.Hkv = Hkv;
    a.Lmax = Lmax;
    a.k = k;
    a.v = v;
    a.rope = rope;
    return launch_kv4(a, B, hd, s);
}

}  // namespace rt
