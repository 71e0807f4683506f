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

#include "rt_internal.h"

#pragma clang fp contract(off)

namespace rt {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
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

// z and h of a group from its extremes, as the cache's dword, in 64 bits up to the roundings:
// a code next to a border must not hang on the order of fp32 operations.  A group with a
// value that is not finite, or whose z or h is not, reads as NaN.
__device__ __forceinline__ unsigned kv4_scale(float lo, float hi, bool finite) {
    const double a = 0.5 * (double)lo, b = 0.5 * (double)hi;
    const unsigned z = bf16_bits((float)(b + a)), h = bf16_bits((float)((b - a) / 15.0));
    const bool ok = finite && (z & 0x7F80u) != 0x7F80u && (h & 0x7F80u) != 0x7F80u;
    return ok ? z << 16 | h : 0x7FC00000u;
}
__device__ __forceinline__ unsigned kv4_code(float x, unsigned s) {
    const double z = (double)kv4_z(s), h = (double)kv4_h(s);
    const double t = h == 0.0 ? 0.0 : ((double)x - z) / h;
    return (unsigned)(int)fmin(fmax(rint((t + 15.0) * 0.5), 0.0), 15.0);
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
        const v4f x1 = *reinterpret_cast<const v4f*>(q + hr * HD + i);
        const v4f x2 = *reinterpret_cast<const v4f*>(q + hr * HD + HALF + i);
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
    for (int r = (t & 127) / TPR; r < kKv4Rows; r += 128 / TPR) {
        const int p = p0 + r;
        const bool in = p >= pos && p < end;
        float x[8];
        const float* src = (is_v ? v : k) + ((size_t)b * M + (in ? p - pos : 0)) * Hkv * HD + (size_t)kh * HD;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = src[8 * o + e];
        if (!is_v) {
            const bool up = 8 * o >= HALF;
            const int i = (8 * o) % HALF;
            const float* other = src + (up ? i : i + HALF);
            const float* cs = rope + ((size_t)(in ? p : 0) * HALF + i) * 2;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double a = x[e], d = other[e], c = cs[2 * e], s = cs[2 * e + 1];
                x[e] = up ? (float)(a * c + d * s) : (float)(a * c - d * s);
            }
        }
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
        const unsigned s = kv4_scale(lo, hi, ((bad >> (lane & 56)) & 0xFFull) == 0ull);
        unsigned word = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) word |= kv4_code(x[e], s) << kv4_shift(e);
        const int P = p % kKv4Block;
        if (is_v) codes[r][o] = word;
        if (in) {
            if (!is_v) reinterpret_cast<unsigned*>(blk)[P * TPR + (o % 8 / 2) * (HD / 32) + o / 8 * 2 + o % 2] = word;
            if (o % 8 == 0) sc[o / 8 * 64 + P] = s;
        }
    }
    __syncthreads();
    // thread (dimension, l): the dword of positions 4 l + (0..3, 8..11) of the 16
    if (t >= 2 * HD) return;
    const int dim = t >> 1, l = t & 1, w = p0 % kKv4Block / 32, s2 = p0 % 32 / 16;
    unsigned word = 0u, mask = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int r = 8 * (e >> 2) + 4 * l + (e & 3), p = p0 + r;
        if (p >= pos && p < end) {
            word |= ((codes[r][dim / 8] >> kv4_shift(dim % 8)) & 15u) << kv4_shift(e);
            mask |= 15u << kv4_shift(e);
        }
    }
    if (mask == 0u) return;
    unsigned* const at = reinterpret_cast<unsigned*>(blk + 32 * HD) +
                         ((dim / 32 * 16 + dim % 16) * 4 + 2 * s2 + l) * 4 + dim % 32 / 16 * 2 + w;
    *at = mask == 0xFFFFFFFFu ? word : (*at & ~mask) | word;
}

// ---- read --------------------------------------------------------------------------------
// Rows (b, m) of K and V as fp32 [B][Hkv][M][HD]; one thread per 8 dimensions of a position
// of K, and per dimension and position of V.
template <int HD>
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint8_t* __restrict__ cache, float* __restrict__ k,
                                                       float* __restrict__ v, int B, int M, int Hkv, int Lmax, int nblk,
                                                       const int* __restrict__ pos_p) {
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;  // (b, kv head, m, dimension)
    const int d = (int)(idx % HD);
    const long long row = idx / HD;
    const int m = (int)(row % M), bh = (int)(row / M);
    if (bh >= B * Hkv) return;
    const int p = kv4_row_pos(pos_p[bh / Hkv], m, Lmax);
    float kx = 0.0f, vx = 0.0f;
    if (p >= 0) {
        const uint8_t* blk = cache + ((size_t)bh * nblk + p / kKv4Block) * kv4_block_bytes(HD);
        const unsigned *w = reinterpret_cast<const unsigned*>(blk), *sc = w + 16 * HD;
        const int P = p % kKv4Block;
        const unsigned kw = w[P * (HD / 8) + (d % 64 / 16) * (HD / 32) + d / 64 * 2 + d % 16 / 8];
        const unsigned vw = w[8 * HD + ((d / 32 * 16 + d % 16) * 4 + P % 32 / 16 * 2 + P % 8 / 4) * 4 + d % 32 / 16 * 2 + P / 32];
        const unsigned ks = sc[d / 64 * 64 + P], vs = sc[HD + d / 64 * 64 + P];
        kx = kv4_z(ks) + kv4_h(ks) * (float)(2 * (int)((kw >> kv4_shift(d % 8)) & 15u) - 15);
        vx = kv4_z(vs) + kv4_h(vs) * (float)(2 * (int)((vw >> kv4_shift(P % 16 / 8 * 4 + P % 4)) & 15u) - 15);
    }
    k[idx] = kx;
    v[idx] = vx;
}

// ---- attention ---------------------------------------------------------------------------
// The eight levels 2 c - 15 of a dword, exact in fp16: a nibble at bits 4..7 of a half under
// 0x6400 is 1024 + 16 c, and (1024 + 16 c) / 8 - 143 = 2 c - 15.
__device__ __forceinline__ v8h kv4_levels(unsigned w) {
    const v2h f = {(_Float16)0.125f, (_Float16)0.125f}, o = {(_Float16)-143.0f, (_Float16)-143.0f};
    v8h r;
    const unsigned n[4] = {w << 4, w, w >> 4, w >> 8};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const v2h x = __builtin_elementwise_fma(__builtin_bit_cast(v2h, (n[i] & 0x00F000F0u) | 0x64006400u), f, o);
        r[2 * i] = x[0];
        r[2 * i + 1] = x[1];
    }
    return r;
}

// x (|x| < 2^15) as two fp16 terms: the error is at most 2^-22 |x| or 2^-25.  The empty asm keeps
// the product that x comes from and its conversion apart: fused (v_fma_mixlo_f16) in one use of
// hi and not in the other, hi differs by its last bit in one of some ten thousand, and that
// much of x was lost (5e-6 of a result over 8192 keys).
__device__ __forceinline__ void kv4_split(v2f x, v2h& hi, v2h& lo) {
    float a = x[0], b = x[1];
    asm("" : "+v"(a), "+v"(b));
    x = v2f{a, b};
    hi = __builtin_convertvector(x, v2h);
    lo = __builtin_convertvector(x - __builtin_convertvector(hi, v2f), v2h);
}
// 2^n as fp32, -126 <= n <= 127
__device__ __forceinline__ float kv4_pow2(int n) { return __uint_as_float((unsigned)(n + 127) << 23); }
__device__ __forceinline__ int kv4_exponent(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 127; }

struct Kv4AttnArgs {
    const float* q;
    const uint8_t* cache;
    float* out;
    float* work;
    const int* pos;
    int M, H, Hkv, Lmax, nblk, tiles, S;
    float scale;  // log2(e) / sqrt(HD)
};

// Rows R = m G + g of KV head kh, 16 a workgroup; lane l works on row l % 16 with the keys of
// lane group h = l / 16.  The split's blocks go to its 4 waves in turn, an online softmax
// (base 2) each:
//   D = U Q^T per group of 64 dimensions (U the keys' levels, exact in fp16; Q two fp16 terms,
//       scaled so that the row's largest is in [2^14, 2^15)),  s = h D + z sum_d q
//   O^T += U^T W^T  (U the values' levels, W = 2^s h, two fp16 terms, scaled by the largest h so far)
//   O   += sum_j 2^s z
// so that all products are exact and all sums fp32.  The waves' results are merged in LDS; with
// S > 1 the split's go to the workspace: O [16][HD], then (m, l) [16][2].
template <int HD>
__global__ void __launch_bounds__(256) kv4_attn_kernel(const Kv4AttnArgs a) {
    constexpr int NG = HD / 64, NT = HD / 16;
    __shared__ float om[4][16][HD + 4];
    __shared__ float ml[4][16][2];
    const int w0 = xcd_order((int)blockIdx.x, (int)gridDim.x);
    const int split = w0 % a.S, unit = w0 / a.S, tile = unit % a.tiles, bh = unit / a.tiles;
    const int b = bh / a.Hkv, kh = bh % a.Hkv, G = a.H / a.Hkv;
    const int t = threadIdx.x, lane = t & 63, i = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int pos = a.pos[b];
    const int R = tile * 16 + i, m = R / G, rows = a.M * G;
    const int last = R < rows ? kv4_row_pos(pos, m, a.Lmax) : -1;  // keys <= last are this row's
    int kend = last + 1;
#pragma unroll
    for (int w = 1; w < 16; w <<= 1) kend = max(kend, __shfl_xor(kend, w, 64));
    kend = __builtin_amdgcn_readfirstlane(kend);
    // the row's queries: dimensions 64 g + 16 h + 8 e + (0..7)
    float qx[NG][16], qs[NG], big = 0.0f;
    const float* qp = a.q + (((size_t)b * a.M + min(m, a.M - 1)) * a.H + (size_t)kh * G + (R < rows ? R % G : 0)) * HD;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const v4f x = *reinterpret_cast<const v4f*>(qp + 64 * g + 16 * h + 4 * e);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                qx[g][4 * e + j] = x[j] * a.scale;
                big = fmaxf(big, fabsf(qx[g][4 * e + j]));
            }
        }
    big = fmaxf(big, __shfl_xor(big, 16, 64));
    big = fmaxf(big, __shfl_xor(big, 32, 64));
    const int qe = min(max(14 - kv4_exponent(big), -113), 126);
    const float qf = kv4_pow2(qe), qi = kv4_pow2(-qe);
    v8h qh[NG][2], ql[NG][2];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        qs[g] = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const v2f x = {qx[g][e] * qf, qx[g][e + 1] * qf};
            v2h hi, lo;
            kv4_split(x, hi, lo);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                qh[g][e / 8][e % 8 + j] = hi[j];
                ql[g][e / 8][e % 8 + j] = lo[j];
                qs[g] += x[j];
            }
        }
        qs[g] += __shfl_xor(qs[g], 16, 64);
        qs[g] += __shfl_xor(qs[g], 32, 64);
    }
    v4f o[NT];
    float zs[NG], mrow = -INFINITY, lrow = 0.0f;
    int ref[NG];  // exponent of the largest h of the values so far
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = v4f{};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        zs[g] = 0.0f;
        ref[g] = -111;
    }
    const uint8_t* const head = a.cache + (size_t)bh * a.nblk * kv4_block_bytes(HD);
    const int nb = (kend + kKv4Block - 1) / kKv4Block;
    for (int j = split * 4 + wave; j < nb; j += 4 * a.S) {
        const uint8_t* blk = head + (size_t)j * kv4_block_bytes(HD);
        const unsigned* sc = reinterpret_cast<const unsigned*>(blk + 64 * HD);
        const int key0 = j * kKv4Block;
        float s[4][4];
        // keys of lane group h in tile (w, x): 32 w + 16 (h / 2) + 8 x + 4 (h % 2) + r
        const int kl = 16 * (h >> 1) + 4 * (h & 1);
#pragma unroll
        for (int wx = 0; wx < 4; ++wx) {
            const int tk = 32 * (wx >> 1) + 8 * (wx & 1);
            unsigned kw[2 * NG];
            const unsigned* kp = reinterpret_cast<const unsigned*>(blk + (tk + 16 * (i >> 3) + (i & 7)) * (HD / 2)) + h * 2 * NG;
            if constexpr (NG == 2) {
                const v4u x = *reinterpret_cast<const v4u*>(kp);
#pragma unroll
                for (int e = 0; e < 4; ++e) kw[e] = x[e];
            } else {
                const v2u x = *reinterpret_cast<const v2u*>(kp);
                kw[0] = x[0];
                kw[1] = x[1];
            }
            v4f dot[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                dot[g] = v4f{};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const v8h u = kv4_levels(kw[2 * g + e]);
                    dot[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(u, qh[g][e], dot[g], 0, 0, 0);
                    dot[g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(u, ql[g][e], dot[g], 0, 0, 0);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[wx][r] = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const v4u x = *reinterpret_cast<const v4u*>(sc + g * 64 + tk + kl);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    s[wx][r] = fmaf(kv4_h(x[r]), dot[g][r], fmaf(kv4_z(x[r]), qs[g], s[wx][r]));
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[wx][r] = key0 + tk + kl + r <= last ? s[wx][r] * qi : -INFINITY;
        }
        float mx = mrow;
#pragma unroll
        for (int wx = 0; wx < 4; ++wx)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[wx][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mb = mx == -INFINITY ? 0.0f : mx;
        const float alpha = exp2f(mrow - mb);
        mrow = mx;
        lrow *= alpha;
#pragma unroll
        for (int wx = 0; wx < 4; ++wx)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[wx][r] = exp2f(s[wx][r] - mb);  // (-inf: 0)
                lrow += s[wx][r];
            }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            v4u vs[4];
            float top = 0.0f;
#pragma unroll
            for (int wx = 0; wx < 4; ++wx) {
                const int tk = 32 * (wx >> 1) + 8 * (wx & 1) + kl;
                vs[wx] = *reinterpret_cast<const v4u*>(sc + HD + g * 64 + tk);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // what lies behind the newest key is not read as a number
                    if (key0 + tk + r >= kend) vs[wx][r] = 0u;
                    top = fmaxf(top, kv4_h(vs[wx][r]));
                }
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const int e = __builtin_amdgcn_readfirstlane(max(ref[g], min(kv4_exponent(top), 127)));
            const float f = kv4_pow2(14 - e), fix = alpha * (ref[g] - e < -126 ? 0.0f : kv4_pow2(ref[g] - e));
            ref[g] = e;
            zs[g] *= alpha;
            v8h wh[2], wl[2];
#pragma unroll
            for (int wx = 0; wx < 4; ++wx) {
                const int tk = 32 * (wx >> 1) + 8 * (wx & 1) + kl;
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    v2h hi, lo;
                    kv4_split(v2f{s[wx][r] * (kv4_h(vs[wx][r]) * f), s[wx][r + 1] * (kv4_h(vs[wx][r + 1]) * f)}, hi, lo);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const bool see = key0 + tk + r + j <= last;
                        wh[wx >> 1][4 * (wx & 1) + r + j] = hi[j];
                        wl[wx >> 1][4 * (wx & 1) + r + j] = lo[j];
                        zs[g] = fmaf(s[wx][r + j], see ? kv4_z(vs[wx][r + j]) : 0.0f, zs[g]);
                    }
                }
            }
#pragma unroll
            for (int u = 2 * g; u < 2 * g + 2; ++u) {
                const v4u x = *reinterpret_cast<const v4u*>(blk + 32 * HD + ((u * 16 + i) * 4 + h) * 16);
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    v4f acc = o[2 * u + v] * fix;
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const v8h lev = kv4_levels(x[2 * v + w]);
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(lev, wh[w], acc, 0, 0, 0);
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(lev, wl[w], acc, 0, 0, 0);
                    }
                    o[2 * u + v] = acc;
                }
            }
        }
    }
    // this wave's O[row][dim], row i, dimensions 32 u + 16 v + 4 h + r
    lrow += __shfl_xor(lrow, 16, 64);
    lrow += __shfl_xor(lrow, 32, 64);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        zs[g] += __shfl_xor(zs[g], 16, 64);
        zs[g] += __shfl_xor(zs[g], 32, 64);
        const float back = kv4_pow2(max(ref[g] - 14, -126));
#pragma unroll
        for (int n = 4 * g; n < 4 * g + 4; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) om[wave][i][n * 16 + 4 * h + r] = fmaf(o[n][r], back, zs[g]);
    }
    if (h == 0) {
        ml[wave][i][0] = mrow;
        ml[wave][i][1] = lrow;
    }
    __syncthreads();
    const int row = t >> 4, RR = tile * 16 + row;
    if (RR >= rows) return;
    float mm = -INFINITY, den = 0.0f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[w][row][0]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = ml[w][row][0] == -INFINITY ? 0.0f : exp2f(ml[w][row][0] - mm);
        den += f[w] * ml[w][row][1];
    }
    float* dst;
    float inv = 1.0f;
    if (a.S > 1) {
        float* part = a.work + ((size_t)unit * a.S + split) * (16 * (HD + 2));
        dst = part + row * HD;
        if ((t & 15) == 0) {
            part[16 * HD + 2 * row] = mm;
            part[16 * HD + 2 * row + 1] = den;
        }
    } else {
        dst = a.out + (((size_t)b * a.M + RR / G) * a.H + (size_t)kh * G + RR % G) * HD;
        inv = den;
    }
#pragma unroll
    for (int d = (t & 15) * 4; d < HD; d += 64) {
        v4f x{};
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = f[w] == 0.0f ? x[j] : x[j] + f[w] * om[w][row][d + j];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = mm == -INFINITY && den == 0.0f ? 0.0f : x[j] / inv;
        *reinterpret_cast<v4f*>(dst + d) = x;
    }
}

// out from the S partials of every unit: one thread per four values.
template <int HD>
__global__ void __launch_bounds__(256) kv4_combine_kernel(const Kv4AttnArgs a, int units) {
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
    const int d = (int)(idx % (HD / 4)) * 4, row = (int)(idx / (HD / 4) % 16);
    const long long unit = idx / (HD / 4) / 16;
    if (unit >= units) return;
    const int G = a.H / a.Hkv, tile = (int)(unit % a.tiles), bh = (int)(unit / a.tiles), R = tile * 16 + row;
    if (R >= a.M * G) return;
    const float* part = a.work + (size_t)unit * a.S * (16 * (HD + 2));
    float mm = -INFINITY, den = 0.0f;
    for (int s = 0; s < a.S; ++s) mm = fmaxf(mm, part[(size_t)s * 16 * (HD + 2) + 16 * HD + 2 * row]);
    v4f x{};
    for (int s = 0; s < a.S; ++s) {
        const float* ps = part + (size_t)s * 16 * (HD + 2);
        const float m = ps[16 * HD + 2 * row], l = ps[16 * HD + 2 * row + 1];
        if (m == -INFINITY && l == 0.0f) continue;
        const float f = exp2f(m - mm);
        const v4f y = *reinterpret_cast<const v4f*>(ps + row * HD + d);
        den += f * l;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] += f * y[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = den == 0.0f ? 0.0f : x[j] / den;
    *reinterpret_cast<v4f*>(a.out + (((size_t)(bh / a.Hkv) * a.M + R / G) * a.H + (size_t)(bh % a.Hkv) * G + R % G) * HD + d) = x;
}

// Workgroups of 256 in one launch: its work items are counted in 32 bits.
constexpr long long kMaxGroups = 0xFFFFFFFFll / 256;

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
    const long long n = ((long long)B * Hkv * M * hd + 255) / 256;
    if (n > kMaxGroups) return hipErrorInvalidValue;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(256), 0, s, static_cast<const uint8_t*>(cache), k, v, B, M,
                           Hkv, Lmax, nblk, pos);
    };
    if (hd == 128) go(kv4_read_kernel<128>);
    else go(kv4_read_kernel<64>);
    return hipGetLastError();
}

namespace {
// Row tiles of 16, and the splits of the keys that fill the chip (two workgroups a CU) where
// the units alone do not.
struct Kv4Shape {
    long long units;
    int tiles, S;
};
Kv4Shape kv4_shape(int B, int M, int H, int Hkv, int Lmax) {
    Kv4Shape p;
    const long long tiles = ((long long)M * (H / Hkv) + 15) / 16;
    p.tiles = (int)std::min(tiles, 0x7FFFFFFFll);
    p.units = (long long)B * Hkv * tiles;
    const int quads = (Lmax + 4 * kKv4Block - 1) / (4 * kKv4Block);
    p.S = (int)std::max(1ll, std::min<long long>(quads, (512 + p.units - 1) / p.units));
    return p;
}
}  // namespace

size_t kv4_attention_workspace(int B, int M, int H, int Hkv, int hd, int Lmax) {
    const Kv4Shape p = kv4_shape(B, M, H, Hkv, Lmax);
    return p.S > 1 ? (size_t)p.units * p.S * 16 * (hd + 2) * sizeof(float) : 0;
}

hipError_t launch_kv4_attention(const float* q, const void* cache, float* out, int B, int M, int H, int Hkv, int hd,
                                int Lmax, const int* pos, float* work, hipStream_t s) {
    const Kv4Shape p = kv4_shape(B, M, H, Hkv, Lmax);
    if (p.units * p.S > kMaxGroups) return hipErrorInvalidValue;
    const Kv4AttnArgs a{q, static_cast<const uint8_t*>(cache), out, work, pos, M, H, Hkv, Lmax,
                        (Lmax + kKv4Block - 1) / kKv4Block, p.tiles, p.S, 1.44269504088896341f / sqrtf((float)hd)};
    auto go = [&](auto kernel, auto combine) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(p.units * p.S)), dim3(256), 0, s, a);
        if (p.S > 1)
            hipLaunchKernelGGL(combine, dim3((unsigned)((p.units * 16 * (hd / 4) + 255) / 256)), dim3(256), 0, s, a,
                               (int)p.units);
    };
    if (hd == 128) go(kv4_attn_kernel<128>, kv4_combine_kernel<128>);
    else go(kv4_attn_kernel<64>, kv4_combine_kernel<64>);
    return hipGetLastError();
}

}  // namespace rt
