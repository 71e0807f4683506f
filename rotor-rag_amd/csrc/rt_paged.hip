// A KV cache in pages, in fp32, bf16 or fp16: RoPE + append, attention of one token a sequence over
// it (with or without accumulating what every slot weighed), both in one call, and eviction by
// accumulated weight.
//
// Callers in the reference: MultiHeadAttention.forward (src/rotor/transformer.py:206-292: KV
// concat :250-252, GQA repeat :260-263, scores/softmax/AV :267-281) with the per-layer cache
// list of BitNetModel.forward (src/rotor/bitnet_model.py:223-228), which grows by copying and is
// never cut.
//
// A layer's cache is K pages and V pages [pages][Hkv][page][HD], page 16 to 256 slots, a power of two.
// Slot t of sequence b is row t % page of page table[b][t / page].  An entry outside [0, pages) is a
// hole: its slots are not there.  Kernels look an entry up before they use it as an address, so no
// table makes them read or write outside the cache.
#include <algorithm>
#include <climits>

#include "rt_internal.h"

namespace rt {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned short v4s __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

namespace {

constexpr long long kPagedMaxGroups = 0x7FFFFFFF;

template <int T>
struct Elem;  // an element of the cache, by RT_PAGED_*
template <>
struct Elem<kPagedF32> {
    typedef float type;
};
template <>
struct Elem<kPagedBf16> {
    typedef unsigned short type;
};
template <>
struct Elem<kPagedF16> {
    typedef unsigned short type;
};

__device__ __forceinline__ unsigned short paged_bf16(float x) {  // to nearest, ties to even; NaN stays one
    const unsigned u = __float_as_uint(x);
    const unsigned r = (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
    return (unsigned short)((u & 0x7FFFFFFFu) > 0x7F800000u ? (u >> 16) | 0x40u : r);
}
template <int T>
__device__ __forceinline__ typename Elem<T>::type paged_round(float x) {
    if constexpr (T == kPagedF32) return x;
    else if constexpr (T == kPagedBf16) return paged_bf16(x);
    else return __builtin_bit_cast(unsigned short, (_Float16)x);
}
// Eight numbers into a row of the cache (16-byte aligned).
template <int T>
__device__ __forceinline__ void paged_store8(typename Elem<T>::type* at, const float (&x)[8]) {
    if constexpr (T == kPagedF32) {
        *reinterpret_cast<v4f*>(at) = v4f{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<v4f*>(at + 4) = v4f{x[4], x[5], x[6], x[7]};
    } else {
        v4u w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (unsigned)paged_round<T>(x[2 * i]) | (unsigned)paged_round<T>(x[2 * i + 1]) << 16;
        *reinterpret_cast<v4u*>(at) = w;
    }
}

// a b - c d of fp32 numbers: exact products and one rounding to 64 bits, one to fp32.  (A difference with one product's rounding
// taken back, in fp32, is within 1.5 units in the last place; but a number next to a border between two bf16
// then rounds to the other one: 3 keys in a million.)
__device__ __forceinline__ float paged_diff(float a, float b, float c, float d) { return (float)((double)a * b - (double)c * d); }
// Dimensions d .. d + 3 (d % 4 == 0) of a row x, rotated over its first `rotary` (a multiple of 8); cs: (cos, sin) of the
// row's position.  Half: pairs (i, i + rotary / 2); interleaved: (2 i, 2 i + 1).
__device__ __forceinline__ v4f paged_rotate4(const float* x, const float* cs, int d, int rotary, bool interleaved) {
    v4f y = *reinterpret_cast<const v4f*>(x + d);
    if (d >= rotary) return y;
    if (interleaved) {
        const v4f c = *reinterpret_cast<const v4f*>(cs + d);  // pairs d / 2, d / 2 + 1
        return v4f{paged_diff(y[0], c[0], y[1], c[1]), paged_diff(y[1], c[0], -y[0], c[1]), paged_diff(y[2], c[2], y[3], c[3]),
                   paged_diff(y[3], c[2], -y[2], c[3])};
    }
    const bool up = d >= rotary / 2;
    const int i = up ? d - rotary / 2 : d;
    const v4f z = *reinterpret_cast<const v4f*>(x + (up ? i : i + rotary / 2));
    const v4f c0 = *reinterpret_cast<const v4f*>(cs + 2 * i), c1 = *reinterpret_cast<const v4f*>(cs + 2 * i + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float c = e < 2 ? c0[2 * e] : c1[2 * e - 4], s = e < 2 ? c0[2 * e + 1] : c1[2 * e - 3];
        y[e] = paged_diff(y[e], c, up ? -z[e] : z[e], s);
    }
    return y;
}

// Where slot t of sequence b lies (elements from the cache's start to the first head's row; kv head h is page * HD * h
// further), or -1: no such slot.
__device__ __forceinline__ long long paged_slot(const PagedCache& c, int HD, int b, int t) {
    if (t < 0 || t >= c.P << c.shift) return -1;
    const int id = c.table[(size_t)b * c.P + (t >> c.shift)];
    if (id < 0 || id >= c.pages) return -1;
    return (long long)id * c.page_stride + (long long)(t & ((1 << c.shift) - 1)) * HD;
}

// ---- append ------------------------------------------------------------------------------
// A thread has 8 dimensions of one head of one row (q heads, then k, then v heads).  A head's threads are in one wave, whose
// loads are all done before its stores, so q_out may be q.  Bound by memory: each number is read and written once (a pair's
// other half comes from the same lines).
template <int T, int HD>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedCache c, PagedNew n, float* q_out, int M, int H) {
    constexpr int L = HD / 8;
    const unsigned units = H + 2 * c.Hkv, per = units * L;
    const unsigned long long first = (unsigned long long)blockIdx.x * 256u;
    const unsigned long long row0 = first / per;
    const unsigned local = (unsigned)(first - row0 * per) + threadIdx.x, skip = local / per;
    const unsigned long long row = row0 + skip;
    if (row >= (unsigned long long)c.B * M) return;
    const unsigned item = local - skip * per;
    const int unit = item / L, o = item % L * 8;
    const int b = (int)(row / (unsigned)M), m = (int)(row - (unsigned long long)b * M);
    const long long p = (long long)n.pos[b] + m, t = (long long)c.lens[b] + m;
    const int count = n.counts ? n.counts[b] : M;
    const long long at = m < count && p >= 0 && p < n.rope_rows && t >= 0 && t <= INT_MAX ? paged_slot(c, HD, b, (int)t) : -1;
    const float* cs = n.rope + (size_t)(at >= 0 ? p : 0) * n.rotary;
    float x[8];
    if (unit < H) {
        const size_t base = ((size_t)row * H + unit) * HD;
        v4f y0{}, y1{};
        if (at >= 0) {
            y0 = paged_rotate4(n.q + base, cs, o, n.rotary, n.interleaved);
            y1 = paged_rotate4(n.q + base, cs, o + 4, n.rotary, n.interleaved);
        }
        *reinterpret_cast<v4f*>(q_out + base + o) = y0;
        *reinterpret_cast<v4f*>(q_out + base + o + 4) = y1;
        return;
    }
    if (at < 0) return;
    const bool is_v = unit >= H + c.Hkv;
    const int kh = unit - H - (is_v ? c.Hkv : 0);
    const size_t base = ((size_t)row * c.Hkv + kh) * HD;
    v4f y0, y1;
    if (is_v) {
        y0 = *reinterpret_cast<const v4f*>(n.v + base + o);
        y1 = *reinterpret_cast<const v4f*>(n.v + base + o + 4);
    } else {
        y0 = paged_rotate4(n.k + base, cs, o, n.rotary, n.interleaved);
        y1 = paged_rotate4(n.k + base, cs, o + 4, n.rotary, n.interleaved);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = y0[e];
        x[4 + e] = y1[e];
    }
    typedef typename Elem<T>::type E;
    E* const cache = static_cast<E*>(c.cache) + (is_v ? c.kv_stride : 0);
    paged_store8<T>(cache + at + ((long long)kh << c.shift) * HD + o, x);
}

// ---- attention ---------------------------------------------------------------------------
// One token a sequence: for every head h, over slots t < n,
//   s_t = log2(e) / sqrt(HD) q_h . k_t,   o_h = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m),   m = max s_t,
// in one pass, the sums so far rescaled wherever m grows.  A workgroup has the up to 16 heads of a
// tile (the query heads of one KV head) and one split of the slots, dealt to its waves in tiles of TK
// slots.  The products run on the matrix cores with 16 columns for the heads:
//   S^T [slots x heads] = K Q^T,   O^T [dimensions x heads] = V^T P^T.
// Lane l is column i = l % 16 with lane group g = l / 16.  A product over 32 (fp32: 4) takes of both operands the numbers
// 8 g .. 8 g + 7 (g) from lane group g, and leaves rows 4 g + r in it; which numbers these are is free, as long as both operands
// agree.  So K goes from memory straight into place (16 bytes of a slot's row a lane); the scores of slots 4 g + r of two row
// tiles, which a lane has then, are its eight of P; and of V, lane group g loads whole rows of those same eight slots, a lane
// HD / 16 dimensions of each, and pairs them by slot with one v_perm a pair: no number passes through LDS.
//
// fp32 numbers times 16-bit ones, in fp32: x is cut into three bf16 that sum up to x exactly (for a cache in
// bf16), or two fp16 and what is left times 2^20 as a third in sums of its own (fp16, x scaled into [0, 2^15]): every product
// is then exact, and all sums are fp32.  Two terms would leave 2^-17 (bf16), or 2^-40 of the row's largest (fp16), which
// numbers 2^16 apart would show.  A cache in fp32 takes fp32 products.
//
// Every load is issued half a round before its use: the next tile's keys when this one's are multiplied, its values after
// this one's.
template <int T, int HD>
struct AttnTile;

// The head's row of q, rotated where the step asks for it, and times log2(e) / sqrt(HD): dimensions d .. d + 3.
__device__ __forceinline__ v4f paged_query4(const PagedAttn& a, const float* q, const float* cs, int d) {
    v4f x = cs ? paged_rotate4(q, cs, d, a.n.rotary, a.n.interleaved) : *reinterpret_cast<const v4f*>(q + d);
    return x * a.scale;
}

// The largest of lanes l, l ^ 16, l ^ 32, l ^ 48; their sum.
__device__ __forceinline__ float paged_max4(float x) {
    v2u y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
    y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float paged_sum4(float x) {
    v2u y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(y[0]) + __uint_as_float(y[1]);
    y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}
// high halves of a (low half of the result) and b
__device__ __forceinline__ unsigned paged_high(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ unsigned paged_low(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }

// Eight fp32 as three bf16 each, whose sum they are: the upper bits as they are, what is left, and again.
__device__ __forceinline__ void paged_split(const float (&x)[8], v4u (&t)[3]) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float u = x[e], v = x[e + 1];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            t[k][e / 2] = paged_high(__float_as_uint(u), __float_as_uint(v));
            u -= __uint_as_float(__float_as_uint(u) & 0xFFFF0000u);
            v -= __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
        }
    }
}
// Eight fp32 (up to 2^15) as two fp16 and 2^20 times the rest as a third.  (The empty asm: the conversion must see the number
// that the rest is taken from, not the product that made it.)
constexpr float kRest = 0x1p20f;
__device__ __forceinline__ void paged_split(const float (&x)[8], v8h (&t)[3]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float u = x[e];
        asm("" : "+v"(u));
        t[0][e] = (_Float16)u;
        float r = u - (float)t[0][e];
        asm("" : "+v"(r));
        t[1][e] = (_Float16)r;
        t[2][e] = (_Float16)((r - (float)t[1][e]) * kRest);
    }
}

// Tiles of 32 slots in 16 bits: two row tiles of 16.
template <int T, int HD>
struct AttnTile {
    static constexpr int TK = 32, NS = 8, NC = HD / 32, NO = HD / 16;  // NS scores a lane; NO sums (of 4 dimensions) a lane
    static constexpr bool F16 = T == kPagedF16;
    typedef unsigned short E;
    v4u k[2][NC];
    unsigned v[8][HD / 32];
    v4u q[3][NC];
    v4f o[NO], rest[F16 ? NO : 1];
    float qi;  // fp16: what the products of q are to be multiplied by

    // base: the tile's two halves of 16 slots
    __device__ __forceinline__ void load_k(const E* base0, const E* base1, int i, int g) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int c = 0; c < NC; ++c) k[tt][c] = *reinterpret_cast<const v4u*>((tt ? base1 : base0) + (i * HD + c * 32 + g * 8));
    }
    __device__ __forceinline__ void load_v(const E* base0, const E* base1, int i, int g) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const E* at = (e < 4 ? base0 : base1) + ((4 * g + (e & 3)) * HD + i * (HD / 16));
            if constexpr (HD == 128) {
                const v4u x = *reinterpret_cast<const v4u*>(at);
#pragma unroll
                for (int w = 0; w < 4; ++w) v[e][w] = x[w];
            } else {
                const v2u x = *reinterpret_cast<const v2u*>(at);
                v[e][0] = x[0];
                v[e][1] = x[1];
            }
        }
    }
    // the lane's slot of score (tt, r), counted in the tile
    static __device__ __forceinline__ int slot(int n, int g) { return 16 * (n >> 2) + 4 * g + (n & 3); }
    // the new row of the tile's slot `at`, from LDS
    __device__ __forceinline__ void put(const E* nk, const E* nv, int at, int i, int g) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
            if (at == 16 * tt + i)
#pragma unroll
                for (int c = 0; c < NC; ++c) k[tt][c] = *reinterpret_cast<const v4u*>(nk + c * 32 + g * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (at == slot(e, g))
#pragma unroll
                for (int w = 0; w < HD / 32; ++w) v[e][w] = reinterpret_cast<const unsigned*>(nv)[i * (HD / 32) + w];
    }
    __device__ __forceinline__ void hide(int n) {  // slot n of the lane's eight is not there
#pragma unroll
        for (int w = 0; w < HD / 32; ++w) v[n][w] = 0u;
    }
    __device__ __forceinline__ void set_query(const PagedAttn& a, const float* row, const float* cs, int g) {
        float x[NC][8], big = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v4f y = paged_query4(a, row, cs, c * 32 + g * 8 + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[c][4 * h + e] = y[e];
                    big = fmaxf(big, fabsf(y[e]));
                }
            }
        if constexpr (F16) {  // the largest into [2^14, 2^15)
            big = paged_max4(big);
            const int n = min(max(14 + 127 - (int)(__float_as_uint(big) >> 23), -113), 126);
            const float f = __uint_as_float((unsigned)(n + 127) << 23);
            qi = __uint_as_float((unsigned)(127 - n) << 23);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[c][e] *= f;
                v8h t[3];
                paged_split(x[c], t);
#pragma unroll
                for (int p = 0; p < 3; ++p) q[p][c] = __builtin_bit_cast(v4u, t[p]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                v4u t[3];
                paged_split(x[c], t);
#pragma unroll
                for (int p = 0; p < 3; ++p) q[p][c] = t[p];
            }
        }
    }
    static __device__ __forceinline__ v4f mul(const v4u& x, const v4u& y, const v4f& z) {
        if constexpr (F16)
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), z, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, x), __builtin_bit_cast(v8b, y), z, 0, 0, 0);
    }
    __device__ __forceinline__ void scores(float (&s)[NS]) {
        v4f d[2] = {}, r[2] = {};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                (F16 ? r : d)[tt] = mul(k[tt][c], q[2][c], (F16 ? r : d)[tt]);
                d[tt] = mul(k[tt][c], q[1][c], d[tt]);
                d[tt] = mul(k[tt][c], q[0][c], d[tt]);
            }
#pragma unroll
        for (int n = 0; n < 8; ++n) s[n] = F16 ? (d[n >> 2][n & 3] + r[n >> 2][n & 3] * (1.0f / kRest)) * qi : d[n >> 2][n & 3];
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < NO; ++j) o[j] = v4f{};
        if constexpr (F16)
#pragma unroll
            for (int j = 0; j < NO; ++j) rest[j] = v4f{};
    }
    __device__ __forceinline__ void scale(float f) {
#pragma unroll
        for (int j = 0; j < NO; ++j) o[j] *= f;
        if constexpr (F16)
#pragma unroll
            for (int j = 0; j < NO; ++j) rest[j] *= f;
    }
    __device__ __forceinline__ void values(float (&p)[NS]) {
        v4u t[3];
        if constexpr (F16) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = p[e] * 0x1p15f;
            v8h y[3];
            paged_split(x, y);
#pragma unroll
            for (int n = 0; n < 3; ++n) t[n] = __builtin_bit_cast(v4u, y[n]);
        } else paged_split(p, t);
#pragma unroll
        for (int j = 0; j < NO; ++j) {
            v4u x;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[e] = j & 1 ? paged_high(v[2 * e][j / 2], v[2 * e + 1][j / 2]) : paged_low(v[2 * e][j / 2], v[2 * e + 1][j / 2]);
            v4f& third = F16 ? rest[j % (F16 ? NO : 1)] : o[j];
            third = mul(x, t[2], third);
            o[j] = mul(x, t[1], o[j]);
            o[j] = mul(x, t[0], o[j]);
        }
    }
    // the lane's sums of dimensions dim(r) .. dim(r) + NO - 1, r = 0..3
    static constexpr int ND = NO, NR = 4;
    static __device__ __forceinline__ int dim(int r, int g) { return (4 * g + r) * NO; }
    __device__ __forceinline__ float out(int r, int j) const {
        if constexpr (F16) return (o[j][r] + rest[j][r] * (1.0f / kRest)) * 0x1p-15f;
        else return o[j][r];
    }
};

// Tiles of 16 slots in fp32.
template <int HD>
struct AttnTile<kPagedF32, HD> {
    static constexpr int TK = 16, NS = 4, NC = HD / 16, NU = HD / 64;
    typedef float E;
    v4f k[NC], v[4][NU], q[NC], o[NU][4];

    __device__ __forceinline__ void load_k(const E* base0, const E*, int i, int g) {
#pragma unroll
        for (int c = 0; c < NC; ++c) k[c] = *reinterpret_cast<const v4f*>(base0 + (i * HD + c * 16 + g * 4));
    }
    __device__ __forceinline__ void load_v(const E* base0, const E*, int i, int g) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int u = 0; u < NU; ++u) v[r][u] = *reinterpret_cast<const v4f*>(base0 + ((4 * g + r) * HD + u * 64 + i * 4));
    }
    static __device__ __forceinline__ int slot(int n, int g) { return 4 * g + n; }
    __device__ __forceinline__ void put(const E* nk, const E* nv, int at, int i, int g) {
        if (at == i)
#pragma unroll
            for (int c = 0; c < NC; ++c) k[c] = *reinterpret_cast<const v4f*>(nk + c * 16 + g * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (at == slot(r, g))
#pragma unroll
                for (int u = 0; u < NU; ++u) v[r][u] = *reinterpret_cast<const v4f*>(nv + u * 64 + i * 4);
    }
    __device__ __forceinline__ void hide(int n) {
#pragma unroll
        for (int u = 0; u < NU; ++u) v[n][u] = v4f{};
    }
    __device__ __forceinline__ void set_query(const PagedAttn& a, const float* row, const float* cs, int g) {
#pragma unroll
        for (int c = 0; c < NC; ++c) q[c] = paged_query4(a, row, cs, c * 16 + g * 4);
    }
    __device__ __forceinline__ void scores(float (&s)[NS]) {
        v4f d[2] = {};  // (two chains: a product waits for the one before it in its own)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int n = 0; n < 4; ++n) d[n & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c][n], q[c][n], d[n & 1], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < 4; ++n) s[n] = d[0][n] + d[1][n];
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int n = 0; n < 4; ++n) o[u][n] = v4f{};
    }
    __device__ __forceinline__ void scale(float f) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int n = 0; n < 4; ++n) o[u][n] *= f;
    }
    __device__ __forceinline__ void values(float (&p)[NS]) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int n = 0; n < 4; ++n) o[u][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][u][n], p[r], o[u][n], 0, 0, 0);
    }
    static constexpr int ND = 4, NR = 4 * NU;
    static __device__ __forceinline__ int dim(int r, int g) { return 64 * (r >> 2) + 4 * (4 * g + (r & 3)); }
    __device__ __forceinline__ float out(int r, int j) const { return o[r >> 2][j][r & 3]; }
};

// Slots that the token of sequence b attends to (STEP: its own, which is put there in this launch, among them).
template <bool STEP>
__device__ __forceinline__ int paged_len(const PagedAttn& a, int b) {
    const int cap = a.c.P << a.c.shift, n = a.c.lens[b];
    if constexpr (STEP) {
        const int p = a.n.pos[b];
        // (a token without a place or an angle is not there, and attends to nothing)
        return p < 0 || p >= a.n.rope_rows || paged_slot(a.c, 0, b, n) < 0 ? 0 : n + 1;
    }
    return min(max(n, 0), cap);
}
// Tiles a split has, for a sequence of `tiles`: as many as fill S splits, but kPagedLeast at least.
__device__ __forceinline__ int paged_piece(int tiles, int S, int least) { return max((tiles + S - 1) / S, least); }

constexpr int kWaves = 4;

template <int T, int HD, bool STEP>
__global__ void __launch_bounds__(64 * kWaves, 2) paged_attn_kernel(PagedAttn a) {
    typedef AttnTile<T, HD> Tile;
    typedef typename Tile::E E;
    constexpr int TK = Tile::TK;
    __shared__ float part[kWaves][16][HD + 4];
    __shared__ float ml[kWaves][16][2];
    __shared__ __align__(16) E fresh[STEP ? 2 : 1][STEP ? HD : 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const int split = blockIdx.x % a.S, unit = blockIdx.x / a.S;  // unit: (b, KV head, tile of heads)
    const int ht = unit % a.tiles, bk = unit / a.tiles, kh = bk % a.c.Hkv, b = bk / a.c.Hkv;
    const int len = paged_len<STEP>(a, b);
    const int tiles = (len + TK - 1) / TK, piece = paged_piece(tiles, a.S, a.least);
    const int first = split * piece, last = min(first + piece, tiles);
    const int rows = min(a.G - 16 * ht, 16);
    if (first >= last && (a.S > 1 || split > 0)) return;
    const int h0 = kh * a.G + 16 * ht;  // the tile's first head
    const int cap = a.c.P << a.c.shift;
    Tile x;
    float m = -INFINITY, l = 0.0f;
    x.clear();
    if (first + wave < last) {
        // the pages of the wave's next 64 tiles, a tile a lane (two where a page is half a tile)
        int id0 = 0, id1 = 0;
        auto look = [&](int t) {
            const int s = (t + lane * kWaves) * TK;
            const int* row = a.c.table + (size_t)b * a.c.P;
            id0 = s < len ? row[s >> a.c.shift] : -1;
            id1 = TK == 32 && s + 16 < len ? row[(s + 16) >> a.c.shift] : -1;
        };
        const E* const kbase = static_cast<const E*>(a.c.cache) + ((long long)kh << a.c.shift) * HD;
        const int in_page = (1 << a.c.shift) - 1;
        auto base = [&](int n, int t, int half, bool& there) {
            const int id = __builtin_amdgcn_readlane(half ? id1 : id0, n & 63);
            there = id >= 0 && id < a.c.pages;
            return kbase + (long long)(there ? id : 0) * a.c.page_stride + ((t * TK + 16 * half) & in_page) * HD;
        };
        look(first + wave);
        int t = first + wave, n = 0;
        bool there0, there1 = false, next0, next1 = false;
        const E* b0 = base(n, t, 0, there0);
        const E* b1 = TK == 32 ? base(n, t, 1, there1) : b0;
        x.load_k(b0, b1, i, g);
        x.load_v(b0 + a.c.kv_stride, b1 + a.c.kv_stride, i, g);
        const int head = h0 + min(i, rows - 1);  // (columns past the last head repeat it)
        const float* cs = STEP ? a.n.rope + (size_t)a.n.pos[b] * a.n.rotary : nullptr;
        x.set_query(a, a.q + ((size_t)b * a.H + head) * HD, cs, g);
        if constexpr (STEP) {
            // the new row: rotated, rounded and written by the wave that has the last tile, which takes it from LDS
            if (last == tiles && (tiles - 1 - first) % kWaves == wave && lane < HD / 4) {
                const bool is_v = lane >= HD / 8;
                const int o = lane % (HD / 8) * 8;
                const float* src = (is_v ? a.n.v : a.n.k) + (size_t)bk * HD;
                const v4f y0 = is_v ? *reinterpret_cast<const v4f*>(src + o) : paged_rotate4(src, cs, o, a.n.rotary, a.n.interleaved);
                const v4f y1 =
                    is_v ? *reinterpret_cast<const v4f*>(src + o + 4) : paged_rotate4(src, cs, o + 4, a.n.rotary, a.n.interleaved);
                const float y[8] = {y0[0], y0[1], y0[2], y0[3], y1[0], y1[1], y1[2], y1[3]};
                paged_store8<T>(&fresh[is_v][o], y);
                if (ht == 0) {
                    E* const cache = static_cast<E*>(a.c.cache) + (is_v ? a.c.kv_stride : 0) + ((long long)kh << a.c.shift) * HD;
                    paged_store8<T>(cache + paged_slot(a.c, HD, b, len - 1) + o, y);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");  // (for the compiler: one wave's LDS accesses are in order)
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
        }
        for (; t < last; t += kWaves, ++n, there0 = next0, there1 = next1) {
            const bool more = t + kWaves < last;
            if constexpr (STEP)
                if (t == tiles - 1) x.put(fresh[0], fresh[1], len - 1 - t * TK, i, g);
            float s[Tile::NS];
            x.scores(s);
            if (more) {
                if (((n + 1) & 63) == 0) look(t + kWaves);
                b0 = base(n + 1, t + kWaves, 0, next0);
                b1 = TK == 32 ? base(n + 1, t + kWaves, 1, next1) : b0;
                x.load_k(b0, b1, i, g);
            }
            if (t == tiles - 1 || !there0 || (TK == 32 && !there1)) {
#pragma unroll
                for (int e = 0; e < Tile::NS; ++e) {
                    const int at = Tile::slot(e, g);
                    if (t * TK + at >= len || !(TK == 32 && e >= 4 ? there1 : there0)) {
                        s[e] = -INFINITY;
                        x.hide(e);
                    }
                }
            }
            if (a.scores && i < rows) {
                float* const to = a.scores + ((size_t)b * a.H + h0 + i) * cap + t * TK;
#pragma unroll
                for (int e = 0; e < Tile::NS; e += 4)
                    if (TK == 16 || t * TK + 16 * (e >> 2) < cap)
                        *reinterpret_cast<v4f*>(to + Tile::slot(e, g)) = v4f{s[e], s[e + 1], s[e + 2], s[e + 3]};
            }
            float top = s[0];
#pragma unroll
            for (int e = 1; e < Tile::NS; ++e) top = fmaxf(top, s[e]);
            top = fmaxf(m, paged_max4(top));
            if (__any(top > m)) {
                const float f = top > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
                x.scale(f);
                l *= f;
                m = top;
            }
            const float ref = m > -INFINITY ? m : 0.0f;
#pragma unroll
            for (int e = 0; e < Tile::NS; ++e) {
                s[e] = __builtin_amdgcn_exp2f(s[e] - ref);
                l += s[e];
            }
            x.values(s);
            if (more) x.load_v(b0 + a.c.kv_stride, b1 + a.c.kv_stride, i, g);
        }
    }
    // the waves' sums, joined
    l = paged_sum4(l);
    if (g == 0) {
        ml[wave][i][0] = m;
        ml[wave][i][1] = l;
    }
    __syncthreads();
    float M = ml[0][i][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, ml[w][i][0]);
    const float ref = M > -INFINITY ? M : 0.0f;
    if (i < rows) {
        const float f = __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
        for (int r = 0; r < Tile::NR; ++r)
#pragma unroll
            for (int j = 0; j < Tile::ND; j += 4)
                *reinterpret_cast<v4f*>(&part[wave][i][Tile::dim(r, g) + j]) =
                    v4f{x.out(r, j) * f, x.out(r, j + 1) * f, x.out(r, j + 2) * f, x.out(r, j + 3) * f};
    }
    __syncthreads();
    for (int e = threadIdx.x * 4; e < rows * HD; e += 64 * kWaves * 4) {
        const int row = e / HD, d = e % HD;
        v4f y = *reinterpret_cast<const v4f*>(&part[0][row][d]);
#pragma unroll
        for (int w = 1; w < kWaves; ++w) y += *reinterpret_cast<const v4f*>(&part[w][row][d]);
        float top = ml[0][row][0], sum = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, ml[w][row][0]);
        const float at = top > -INFINITY ? top : 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += ml[w][row][1] * __builtin_amdgcn_exp2f(ml[w][row][0] - at);
        if (a.S == 1) {
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;  // (no slot: zeros)
            *reinterpret_cast<v4f*>(a.out + ((size_t)b * a.H + h0 + row) * HD + d) = y * inv;
        } else *reinterpret_cast<v4f*>(a.part + (((size_t)unit * a.S + split) * 16 + row) * HD + d) = y;
        if ((a.S > 1 || a.scores) && d == 0)
            *reinterpret_cast<v2f*>(a.ml + (((size_t)unit * a.S + split) * 16 + row) * 2) = v2f{top, sum};
    }
}

// The join: workgroups [0, B H): a head's partials into its output; the others: what 1024 slots of a KV head weighed
// (every head's score against its reference and sum), added to the accumulated weights.
template <int HD, bool STEP>
__global__ void __launch_bounds__(256) paged_join_kernel(PagedAttn a, int TK, int joins, int chunks) {
    __shared__ float sums[256 / (HD / 4)][HD];
    const int t = threadIdx.x;
    if ((int)blockIdx.x < joins) {
        const int head = blockIdx.x % a.H, b = blockIdx.x / a.H, kh = head / a.G, in = head % a.G;
        const int tiles = (paged_len<STEP>(a, b) + TK - 1) / TK, piece = paged_piece(tiles, a.S, a.least);
        const int n = (tiles + piece - 1) / piece;
        const size_t first = ((size_t)(b * a.c.Hkv + kh) * a.tiles + in / 16) * a.S;
        const float* ml = a.ml + (first * 16 + in % 16) * 2;
        const float* part = a.part + (first * 16 + in % 16) * HD;
        const int d = t % (HD / 4) * 4, grp = t / (HD / 4);
        float top = -INFINITY;
        for (int s = 0; s < n; ++s) top = fmaxf(top, ml[s * 32]);
        const float ref = top > -INFINITY ? top : 0.0f;
        float sum = 0.0f;
        for (int s = 0; s < n; ++s) sum += ml[s * 32 + 1] * __builtin_amdgcn_exp2f(ml[s * 32] - ref);
        v4f y{};
        for (int s = grp; s < n; s += 256 / (HD / 4))
            y += *reinterpret_cast<const v4f*>(part + (size_t)s * 16 * HD + d) * __builtin_amdgcn_exp2f(ml[s * 32] - ref);
        *reinterpret_cast<v4f*>(&sums[grp][d]) = y;
        __syncthreads();
        if (grp) return;
#pragma unroll
        for (int w = 1; w < 256 / (HD / 4); ++w) y += *reinterpret_cast<const v4f*>(&sums[w][d]);
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        *reinterpret_cast<v4f*>(a.out + ((size_t)b * a.H + head) * HD + d) = y * inv;
        return;
    }
    const int chunk = ((int)blockIdx.x - joins) % chunks, bk = ((int)blockIdx.x - joins) / chunks, b = bk / a.c.Hkv, kh = bk % a.c.Hkv;
    const int len = paged_len<STEP>(a, b), cap = a.c.P << a.c.shift, s0 = chunk * 1024 + t * 4;
    if (chunk * 1024 >= len) return;
    const int tiles = (len + TK - 1) / TK, piece = paged_piece(tiles, a.S, a.least), n = (tiles + piece - 1) / piece;
    v4f add{};
    for (int in = 0; in < a.G; ++in) {
        const float* ml = a.ml + (((size_t)bk * a.tiles + in / 16) * a.S * 16 + in % 16) * 2;
        float top = -INFINITY;
        for (int s = 0; s < n; ++s) top = fmaxf(top, ml[s * 32]);
        const float ref = top > -INFINITY ? top : 0.0f;
        float sum = 0.0f;
        for (int s = 0; s < n; ++s) sum += ml[s * 32 + 1] * __builtin_amdgcn_exp2f(ml[s * 32] - ref);
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        if (s0 < cap) {
            const v4f s = *reinterpret_cast<const v4f*>(a.scores + ((size_t)b * a.H + kh * a.G + in) * cap + s0);
#pragma unroll
            for (int e = 0; e < 4; ++e) add[e] += s0 + e < len ? __builtin_amdgcn_exp2f(s[e] - ref) * inv : 0.0f;
        }
    }
    float* const w = a.weights + (size_t)bk * a.slots + s0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (s0 + e < len) w[e] += add[e];
}

// ---- eviction ----------------------------------------------------------------------------
// Which slots are kept: the last `recent`, and of those before them the largest weights, ties to the lowest slot; slots in
// holes are not there.  One workgroup a KV head of a sequence.  Weights as whole numbers of the same order (NaN above all, -0 as
// 0); the smallest that is kept is found bit by bit, eleven, eleven and ten at a time, from a histogram in LDS; then every
// wave counts its own run of slots, and writes out those that are kept behind those of the waves before it.
constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64;

__device__ __forceinline__ unsigned evict_key(float w) {  // 1 and up (0: not there)
    unsigned u = __float_as_uint(w);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
    if (u == 0x80000000u) u = 0u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ int evict_scan(int x) {  // inclusive, over the lanes
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15, 31
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return x;
}

__global__ void __launch_bounds__(kEvictThreads) paged_select_kernel(PagedEvict a) {
    __shared__ int hist[2048];
    __shared__ int totals[kEvictWaves][2], found[4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int bk = blockIdx.x, b = bk / a.c.Hkv;
    const int cap = a.c.P << a.c.shift, len = min(max(a.c.lens[b], 0), cap);
    const int old = max(len - a.recent, 0);  // slots that are judged; [old, len) stay
    const float* const w = a.weights + (size_t)bk * a.slots;
    const int* const row = a.c.table + (size_t)b * a.c.P;
    auto there = [&](int s) {
        const int id = row[s >> a.c.shift];
        return id >= 0 && id < a.c.pages;
    };
    auto key = [&](int s) { return there(s) ? evict_key(w[s]) : 0u; };
    // the recent ones that are there, and the judged ones
    if (t < 4) found[t] = 0;
    __syncthreads();
    {
        int n = 0, r = 0;
        for (int s = t; s < len; s += kEvictThreads) (s < old ? n : r) += there(s) ? 1 : 0;
        n = evict_scan(n);
        r = evict_scan(r);
        if (lane == 63) {
            atomicAdd(&found[0], n);
            atomicAdd(&found[1], r);
        }
    }
    __syncthreads();
    const int judged = found[0], stay = found[1];
    int want = min(judged, a.keep - stay);  // of the judged ones (recent <= keep)
    // the key of number `want`, counted from the largest: `prefix`; `want` of those equal to it are kept
    unsigned prefix = 0u, mask = 0u;
    if (want > 0 && want < judged) {
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
            for (int n = t; n < 2048; n += kEvictThreads) hist[n] = 0;
            __syncthreads();
            for (int s = t; s < old; s += kEvictThreads) {
                const unsigned k = key(s);
                if (k && (k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
            }
            __syncthreads();
            // from the largest bin down: two bins a thread
            const int hi = bins - 1 - 2 * t, n0 = hi >= 0 ? hist[hi] : 0, n1 = hi >= 1 ? hist[hi - 1] : 0;
            const int incl = evict_scan(n0 + n1);
            if (lane == 63) totals[wave][0] = incl;
            __syncthreads();
            int before = incl - n0 - n1;
            for (int v = 0; v < wave; ++v) before += totals[v][0];
            if (n0 && before < want && before + n0 >= want) {
                found[2] = hi;
                found[3] = want - before;
            } else if (n1 && before + n0 < want && before + n0 + n1 >= want) {
                found[2] = hi - 1;
                found[3] = want - before - n0;
            }
            __syncthreads();
            prefix |= (unsigned)found[2] << shift;
            mask |= (unsigned)(bins - 1) << shift;
            want = found[3];
            __syncthreads();
        }
    } else {  // all of them, or none
        prefix = want > 0 ? 0u : 0xFFFFFFFFu;
        want = 0;
    }
    // every wave has a run of slots
    const int per = (len + kEvictThreads - 1) / kEvictThreads * 64, s0 = wave * per, s1 = min(s0 + per, len);
    auto state = [&](int s, int& more, int& same) {
        const bool in = s < s1;
        const unsigned k = in && s < old ? key(s) : 0u;
        more = (in && s >= old && there(s)) || k > prefix ? 1 : 0;
        same = k && k == prefix ? 1 : 0;
    };
    int above = 0, equal = 0;
    for (int s = s0 + lane; s - lane < s1; s += 64) {
        int more, same;
        state(s, more, same);
        above += more;
        equal += same;
    }
    above = evict_scan(above);
    equal = evict_scan(equal);
    if (lane == 63) {
        totals[wave][0] = above;
        totals[wave][1] = equal;
    }
    __syncthreads();
    above = equal = 0;
    int all = 0;
    int equals = 0;
    for (int v = 0; v < kEvictWaves; ++v) {
        if (v == wave) {
            above = all;
            equal = equals;
        }
        all += totals[v][0];
        equals += totals[v][1];
    }
    int out = above + min(equal, want);  // slots kept before this wave's
    int* const kept = a.kept + (size_t)bk * a.keep;
    float* const left = a.new_weights + (size_t)bk * a.slots;
    for (int s = s0 + lane; s - lane < s1; s += 64) {
        int more, same;
        state(s, more, same);
        const unsigned long long below = (1ull << lane) - 1, ge = __ballot(same);
        const int rank = equal + __popcll(ge & below);  // of an equal one among the equal ones
        const bool keep = more || (same && rank < want);
        const unsigned long long gk = __ballot(keep);
        if (keep) {
            const int at = out + __popcll(gk & below);
            kept[at] = s;
            left[at] = w[s];
        }
        equal += __popcll(ge);
        out += __popcll(gk);
    }
    const int total = all + min(equals, want);
    for (int n = total + t; n < a.keep; n += kEvictThreads) kept[n] = -1;
    for (int n = total + t; n < a.slots; n += kEvictThreads) left[n] = 0.0f;
    if (bk % a.c.Hkv == 0 && t == 0) a.new_lens[b] = total;  // (the same for every head: holes are the sequence's)
}

// The rows of the kept slots, in order, into the new table's pages: 16 bytes a thread of K and of V.
__global__ void __launch_bounds__(256) paged_move_kernel(PagedEvict a, int row_bytes, int esize) {
    const int lanes = row_bytes / 16, rows = 256 / lanes, t = threadIdx.x;
    const int chunks = (a.keep + rows - 1) / rows, chunk = blockIdx.x % chunks, bk = blockIdx.x / chunks;
    const int b = bk / a.c.Hkv, kh = bk % a.c.Hkv, n = chunk * rows + t / lanes, o = t % lanes * 16;
    if (n >= a.keep) return;
    const int s = a.kept[(size_t)bk * a.keep + n];
    if (s < 0) return;
    const int in_page = (1 << a.c.shift) - 1;
    const int from = a.c.table[(size_t)b * a.c.P + (s >> a.c.shift)], to = a.new_table[(size_t)b * a.new_P + (n >> a.c.shift)];
    if (from < 0 || from >= a.c.pages || to < 0 || to >= a.c.pages) return;
    char* const base = static_cast<char*>(a.c.cache) + ((long long)kh << a.c.shift) * row_bytes + o;
    const long long src = (long long)from * a.c.page_stride * esize + (long long)(s & in_page) * row_bytes;
    const long long dst = (long long)to * a.c.page_stride * esize + (long long)(n & in_page) * row_bytes;
    const long long v = a.c.kv_stride * esize;
    const v4u x = *reinterpret_cast<const v4u*>(base + src), y = *reinterpret_cast<const v4u*>(base + src + v);
    *reinterpret_cast<v4u*>(base + dst) = x;
    *reinterpret_cast<v4u*>(base + dst + v) = y;
}

template <typename F>
void paged_by_type(int type, int hd, F go) {
    if (type == kPagedF32) hd == 128 ? go(std::integral_constant<int, kPagedF32>(), std::integral_constant<int, 128>())
                                     : go(std::integral_constant<int, kPagedF32>(), std::integral_constant<int, 64>());
    else if (type == kPagedBf16) hd == 128 ? go(std::integral_constant<int, kPagedBf16>(), std::integral_constant<int, 128>())
                                           : go(std::integral_constant<int, kPagedBf16>(), std::integral_constant<int, 64>());
    else hd == 128 ? go(std::integral_constant<int, kPagedF16>(), std::integral_constant<int, 128>())
                   : go(std::integral_constant<int, kPagedF16>(), std::integral_constant<int, 64>());
}

// Splits, and the tiles a split has at least.
struct PagedShape {
    long long units;
    int tiles, S, least;
};
PagedShape paged_shape(int B, int H, int Hkv, int cap, int type) {
    PagedShape p;
    const int G = H / Hkv, tk = type == kPagedF32 ? 16 : 32;
    p.tiles = (G + 15) / 16;
    p.units = (long long)B * Hkv * p.tiles;
    p.least = kWaves;
    const int most = (cap + tk * p.least - 1) / (tk * p.least);
    p.S = (int)std::max(1ll, std::min<long long>(most, 1024 / p.units));
    return p;
}

}  // namespace

hipError_t launch_paged_append(const PagedCache& c, const PagedNew& n, float* q_out, int M, int H, int type, int hd, hipStream_t s) {
    const unsigned long long items = (unsigned long long)c.B * M * (H + 2 * c.Hkv) * (hd / 8);
    if ((items + 255) / 256 > (unsigned long long)kPagedMaxGroups) return hipErrorInvalidValue;
    paged_by_type(type, hd, [&](auto T, auto HD) {
        hipLaunchKernelGGL((paged_append_kernel<decltype(T)::value, decltype(HD)::value>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0,
                           s, c, n, q_out, M, H);
    });
    return hipGetLastError();
}

// The workspace: partials [unit][S][16][hd], (reference, sum) [unit][S][16][2], scores [B][H][cap], all fp32.
size_t paged_attention_workspace(int B, int H, int Hkv, int cap, int type, int hd, bool weights) {
    const PagedShape p = paged_shape(B, H, Hkv, cap, type);
    const size_t parts = (size_t)p.units * p.S * 16;
    return 4 * ((p.S > 1 ? parts * hd : 0) + (p.S > 1 || weights ? parts * 2 : 0) + (weights ? (size_t)B * H * cap : 0));
}

hipError_t launch_paged_attention(PagedAttn a, bool step, int type, int hd, void* work, hipStream_t s) {
    const int cap = a.c.P << a.c.shift, TK = type == kPagedF32 ? 16 : 32;
    const PagedShape p = paged_shape(a.c.B, a.H, a.c.Hkv, cap, type);
    a.G = a.H / a.c.Hkv;
    a.tiles = p.tiles;
    a.S = p.S;
    a.least = p.least;
    a.scale = 1.44269504088896341f / sqrtf((float)hd);
    const size_t parts = (size_t)p.units * p.S * 16;
    a.part = static_cast<float*>(work);
    a.ml = a.part + (p.S > 1 ? parts * hd : 0);
    a.scores = a.weights ? a.ml + parts * 2 : nullptr;
    const long long groups = p.units * p.S, joins = p.S > 1 ? (long long)a.c.B * a.H : 0;
    const int chunks = a.weights ? (cap + 1023) / 1024 : 0;
    const long long second = joins + (long long)a.c.B * a.c.Hkv * chunks;
    if (groups > kPagedMaxGroups || second > kPagedMaxGroups) return hipErrorInvalidValue;
    paged_by_type(type, hd, [&](auto T, auto HD) {
        constexpr int t = decltype(T)::value, d = decltype(HD)::value;
        if (step) hipLaunchKernelGGL((paged_attn_kernel<t, d, true>), dim3((unsigned)groups), dim3(64 * kWaves), 0, s, a);
        else hipLaunchKernelGGL((paged_attn_kernel<t, d, false>), dim3((unsigned)groups), dim3(64 * kWaves), 0, s, a);
        if (!second) return;
        if (step) hipLaunchKernelGGL((paged_join_kernel<d, true>), dim3((unsigned)second), dim3(256), 0, s, a, TK, (int)joins, chunks);
        else hipLaunchKernelGGL((paged_join_kernel<d, false>), dim3((unsigned)second), dim3(256), 0, s, a, TK, (int)joins, chunks);
    });
    return hipGetLastError();
}

hipError_t launch_paged_evict(const PagedEvict& a, int type, int hd, hipStream_t s) {
    const int esize = type == kPagedF32 ? 4 : 2, row = hd * esize, rows = 256 / (row / 16);
    const long long heads = (long long)a.c.B * a.c.Hkv, moves = heads * ((a.keep + rows - 1) / rows);
    if (moves > kPagedMaxGroups) return hipErrorInvalidValue;
    hipLaunchKernelGGL(paged_select_kernel, dim3((unsigned)heads), dim3(kEvictThreads), 0, s, a);
    hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)moves), dim3(256), 0, s, a, row, esize);
    return hipGetLastError();
}

}  // namespace rt
