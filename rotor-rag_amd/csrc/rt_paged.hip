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
#include <time.h>
#include <unistd.h>

#include <algorithm>
#include <atomic>
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
// Four numbers into a row of the cache.
template <int T>
__device__ __forceinline__ void paged_store4(typename Elem<T>::type* at, const v4f& x) {
    if constexpr (T == kPagedF32) *reinterpret_cast<v4f*>(at) = x;
    else *reinterpret_cast<v4s*>(at) = v4s{paged_round<T>(x[0]), paged_round<T>(x[1]), paged_round<T>(x[2]), paged_round<T>(x[3])};
}

// a b - c d of fp32 numbers: exact products and one rounding to 64 bits, one to fp32.  (A difference with one product's rounding
// taken back, in fp32, is within 1.5 units in the last place; but a number next to a border between two bf16
// then rounds to the other one: 3 keys in a million.)
__device__ __forceinline__ float paged_diff(float a, float b, float c, float d) { return (float)((double)a * b - (double)c * d); }
// Dimensions d .. d + 3 (d % 4 == 0) of a row x, rotated over its first `rotary` (a multiple of 8); cs: (cos, sin) of the
// row's position.  Half: pairs (i, i + rotary / 2); interleaved: (2 i, 2 i + 1).
__device__ __forceinline__ v4f paged_turn_pairs(v4f y, v4f c) {  // (y0, y1), (y2, y3) by (c0, c1), (c2, c3)
    return v4f{paged_diff(y[0], c[0], y[1], c[1]), paged_diff(y[1], c[0], -y[0], c[1]), paged_diff(y[2], c[2], y[3], c[3]),
               paged_diff(y[3], c[2], -y[2], c[3])};
}
__device__ __forceinline__ v4f paged_rotate4(const float* x, const float* cs, int d, int rotary, bool interleaved) {
    v4f y = *reinterpret_cast<const v4f*>(x + d);
    if (d >= rotary) return y;
    if (interleaved) return paged_turn_pairs(y, *reinterpret_cast<const v4f*>(cs + d));
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
// Both fours of a row that item o of HD / 8 has: a pair's two halves where pairs lie apart, else eight in a row.
__device__ __forceinline__ int2 paged_fours(int o, int rotary, bool interleaved) {
    return !interleaved && 8 * o < rotary ? make_int2(4 * o, 4 * o + rotary / 2) : make_int2(8 * o, 8 * o + 4);
}
__device__ __forceinline__ void paged_rotate8(v4f& x, v4f& y, const float* cs, int o, int rotary, bool interleaved) {
    if (8 * o >= rotary) return;
    const v4f c0 = *reinterpret_cast<const v4f*>(cs + 8 * o), c1 = *reinterpret_cast<const v4f*>(cs + 8 * o + 4);
    if (interleaved) {
        x = paged_turn_pairs(x, c0);
        y = paged_turn_pairs(y, c1);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // (the turn of paged_rotate4, pair by pair)
        const float c = e < 2 ? c0[2 * e] : c1[2 * e - 4], s = e < 2 ? c0[2 * e + 1] : c1[2 * e - 3];
        const float u = paged_diff(x[e], c, y[e], s);
        y[e] = paged_diff(y[e], c, -x[e], s);
        x[e] = u;
    }
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
// A thread has 8 dimensions of one head of one row (q heads, then k, then v heads), both halves of its pairs: each number is read
// and written once, by one thread, so q_out may be q.  Bound by memory: 8 prompts of up to 2048 tokens (20 heads over 5 of
// 128, bf16), one call after the other, 77.5 us, 5.25 TB/s; with the
// queries' stores through the caches 88.
template <int T, int HD>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedCache c, PagedNew n, float* q_out, int M, int H) {
    constexpr int L = HD / 8;
    typedef typename Elem<T>::type E;
    const unsigned units = H + 2 * c.Hkv, per = units * L;
    const unsigned long long first = (unsigned long long)blockIdx.x * 256u;
    const unsigned long long row0 = first / per;
    const unsigned local = (unsigned)(first - row0 * per) + threadIdx.x, skip = local / per;
    const unsigned long long row = row0 + skip;
    if (row >= (unsigned long long)c.B * M) return;
    const unsigned item = local - skip * per;
    const int unit = item / L, o = item % L;
    const bool is_q = unit < H, is_v = unit >= H + c.Hkv;
    const int kh = unit - H - (is_v ? c.Hkv : 0);
    const int2 d = is_v ? make_int2(8 * o, 8 * o + 4) : paged_fours(o, n.rotary, n.interleaved);
    const float* const src = is_q ? n.q + ((size_t)row * H + unit) * HD : (is_v ? n.v : n.k) + ((size_t)row * c.Hkv + kh) * HD;
    v4f x = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(src + d.x));
    v4f y = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(src + d.y));
    const int b = (int)(row / (unsigned)M), m = (int)(row - (unsigned long long)b * M);
    const long long p = (long long)n.pos[b] + m, t = (long long)c.lens[b] + m;
    const int count = n.counts ? n.counts[b] : M;
    const long long at = m < count && p >= 0 && p < n.rope_rows && t >= 0 && t <= INT_MAX ? paged_slot(c, HD, b, (int)t) : -1;
    if (at >= 0 && !is_v) paged_rotate8(x, y, n.rope + (size_t)p * n.rotary, o, n.rotary, n.interleaved);
    if (is_q) {
        float* const to = q_out + ((size_t)row * H + unit) * HD;
        __builtin_nontemporal_store(at >= 0 ? x : v4f{}, reinterpret_cast<v4f*>(to + d.x));
        __builtin_nontemporal_store(at >= 0 ? y : v4f{}, reinterpret_cast<v4f*>(to + d.y));
    } else if (at >= 0) {
        E* const to = static_cast<E*>(c.cache) + (is_v ? c.kv_stride : 0) + at + ((long long)kh << c.shift) * HD;
        paged_store4<T>(to + d.x, x);
        paged_store4<T>(to + d.y, y);
    }
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
// is then exact, and all sums are fp32.  Two terms would leave up to 2^-15 of x (bf16, cut off and not rounded), or 2^-40 of the row's
// largest (fp16).  A cache in fp32 takes fp32 products.
//
// Every load is issued half a round before its use: the next tile's keys when this one's are multiplied, its values after
// this one's.
template <int T, int HD, bool ONCE>
struct AttnTile;

// A load of numbers that no other workgroup reads goes past the caches (launch_paged_attention has the measure).
template <bool ONCE, typename V, typename E>
__device__ __forceinline__ V paged_load(const E* at) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const V*>(at));
    else return *reinterpret_cast<const V*>(at);
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

__device__ __forceinline__ void paged_split_bf16(v4f x, v2u (&t)[3]) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        t[k] = v2u{paged_high(__float_as_uint(x[0]), __float_as_uint(x[1])), paged_high(__float_as_uint(x[2]), __float_as_uint(x[3]))};
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] -= __uint_as_float(__float_as_uint(x[e]) & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void paged_split(v4f x, v2u (&t)[3]) {
    unsigned short h[3][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float u = x[e];
        asm("" : "+v"(u));
        const _Float16 a = (_Float16)u;
        float r = u - (float)a;
        asm("" : "+v"(r));
        const _Float16 b = (_Float16)r;
        h[0][e] = __builtin_bit_cast(unsigned short, a);
        h[1][e] = __builtin_bit_cast(unsigned short, b);
        h[2][e] = __builtin_bit_cast(unsigned short, (_Float16)((r - (float)b) * kRest));
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) t[k] = v2u{h[k][0] | (unsigned)h[k][1] << 16, h[k][2] | (unsigned)h[k][3] << 16};
}

// Tiles of 32 slots in 16 bits: two row tiles of 16.
template <int T, int HD, bool ONCE>
struct AttnTile {
    static constexpr int TK = 32, NS = 8, NC = HD / 32, NO = HD / 16;  // NS scores a lane; NO sums (of 4 dimensions) a lane
    static constexpr bool F16 = T == kPagedF16;
    typedef unsigned short E;
    v4u k[2][NC];
    unsigned v[8][HD / 32];
    v4u q[3][NC];
    v4f o[NO], rest[F16 ? NO : 1];
    float qi;  // what a score's products are to be multiplied by: log2(e) / sqrt(HD) and, in fp16, the queries' power of two

    // base: the tile's two halves of 16 slots
    __device__ __forceinline__ void load_k(const E* base0, const E* base1, int i, int g) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
            for (int c = 0; c < NC; ++c) k[tt][c] = paged_load<ONCE, v4u>((tt ? base1 : base0) + (i * HD + c * 32 + g * 8));
    }
    __device__ __forceinline__ void load_v(const E* base0, const E* base1, int i, int g) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const E* at = (e < 4 ? base0 : base1) + ((4 * g + (e & 3)) * HD + i * (HD / 16));
            if constexpr (HD == 128) {
                const v4u x = paged_load<ONCE, v4u>(at);
#pragma unroll
                for (int w = 0; w < 4; ++w) v[e][w] = x[w];
            } else {
                const v2u x = paged_load<ONCE, v2u>(at);
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
    // Queries pass through LDS in the order that lanes take them, [term][c][g][i] of 16 bytes: put by the workgroup, four
    // dimensions a thread (x: of head i, dimensions d .. d + 3; 2^n times that in fp16), taken by every wave.
    static constexpr int QBYTES = 3 * NC * 64 * 16;
    static __device__ __forceinline__ void stage(char* to, v4f x, int i, int d, int n) {
        char* const at = to + ((d / 32 * 4 + d / 8 % 4) * 16 + i) * 16 + d % 8 * 2;
        v2u t[3];
        if constexpr (F16) {
            const float f = __uint_as_float((unsigned)(n + 127) << 23);
            paged_split(v4f{x[0] * f, x[1] * f, x[2] * f, x[3] * f}, t);
        } else paged_split_bf16(x, t);
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<v2u*>(at + p * NC * 1024) = t[p];
    }
    __device__ __forceinline__ void take(const char* from, int n, float scale, int i, int g) {
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int c = 0; c < NC; ++c) q[p][c] = *reinterpret_cast<const v4u*>(from + (((p * NC + c) * 4 + g) * 16 + i) * 16);
        qi = scale * __uint_as_float((unsigned)(127 - n) << 23);
    }
    static __device__ __forceinline__ v4f mul(const v4u& x, const v4u& y, const v4f& z) {
        if constexpr (F16)
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, y), z, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, x), __builtin_bit_cast(v8b, y), z, 0, 0, 0);
    }
    __device__ __forceinline__ void scores(float (&s)[NS]) {
        v4f d[2] = {}, e[2] = {}, r[2] = {};  // (the small terms in sums of their own: fewer roundings of the large one)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                (F16 ? r : e)[tt] = mul(k[tt][c], q[2][c], (F16 ? r : e)[tt]);
                e[tt] = mul(k[tt][c], q[1][c], e[tt]);
                d[tt] = mul(k[tt][c], q[0][c], d[tt]);
            }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const float small = e[n >> 2][n & 3];
            s[n] = (d[n >> 2][n & 3] + (F16 ? small + r[n >> 2][n & 3] * (1.0f / kRest) : small)) * qi;
        }
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
template <int HD, bool ONCE>
struct AttnTile<kPagedF32, HD, ONCE> {
    static constexpr int TK = 16, NS = 4, NC = HD / 16, NU = HD / 64;
    static constexpr bool F16 = false;
    typedef float E;
    v4f k[NC], v[4][NU], q[NC], o[NU][4];
    float qi;

    __device__ __forceinline__ void load_k(const E* base0, const E*, int i, int g) {
#pragma unroll
        for (int c = 0; c < NC; ++c) k[c] = paged_load<ONCE, v4f>(base0 + (i * HD + c * 16 + g * 4));
    }
    __device__ __forceinline__ void load_v(const E* base0, const E*, int i, int g) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int u = 0; u < NU; ++u) v[r][u] = paged_load<ONCE, v4f>(base0 + ((4 * g + r) * HD + u * 64 + i * 4));
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
    static constexpr int QBYTES = NC * 64 * 16;
    static __device__ __forceinline__ void stage(char* to, v4f x, int i, int d, int) {
        *reinterpret_cast<v4f*>(to + ((d / 16 * 4 + d / 4 % 4) * 16 + i) * 16) = x;
    }
    __device__ __forceinline__ void take(const char* from, int, float scale, int i, int g) {
        qi = scale;
#pragma unroll
        for (int c = 0; c < NC; ++c) q[c] = *reinterpret_cast<const v4f*>(from + ((c * 4 + g) * 16 + i) * 16);
    }
    __device__ __forceinline__ void scores(float (&s)[NS]) {
        v4f d[4] = {};  // (four chains: a product waits for the one before it in its own, and long sums lose more)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int n = 0; n < 4; ++n) d[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c][n], q[c][n], d[n], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < 4; ++n) s[n] = ((d[0][n] + d[1][n]) + (d[2][n] + d[3][n])) * qi;
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

// Slots that a sequence of `len` attends to, the step's token among them: should that turn out to have no place or no angle, it
// attends to none, but its share of the launch is as if it had.
template <bool STEP>
__device__ __forceinline__ int paged_span(const PagedAttn& a, int len) {
    const int cap = a.c.P << a.c.shift;
    if constexpr (STEP) return len < 0 || len >= cap ? 0 : len + 1;
    return min(max(len, 0), cap);
}
// The page of a step's token whose slot is the last of `span`, or -1 where it attends to nothing.
__device__ __forceinline__ int paged_newest(const PagedAttn& a, int b, int span) {
    const int p = a.n.pos[b], id = span > 0 ? a.c.table[(size_t)b * a.c.P + ((span - 1) >> a.c.shift)] : -1;
    return p < 0 || p >= a.n.rope_rows || id >= a.c.pages ? -1 : id;
}
__device__ __forceinline__ int paged_scan(int x) {  // inclusive, over the lanes
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15, 31
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return x;
}

// Slots in whole tiles.
__host__ __device__ __forceinline__ int paged_even(int cap) { return (cap + 31) & ~31; }

// The pieces of a launch.  A sequence of n tiles is cut, for each of its `per` units (a KV head's tile of heads), into pieces
// of at most q tiles (one at least), as equal as they can be, q about the least for which all fit the launch's workgroups.  The first
// B per places have the units' first pieces; the others the further ones, in the order (sequence, KV head, piece, tile of heads).
// Every wave works this out for itself, lane b for sequence b: the host does not know the lengths, and with the same number of
// pieces for each the longest sequence decides the launch.
// Tiles of heads that read the same keys, which stand next to each other in that order, go to one of the 8 dies (workgroup
// number mod 8), whose L2 then reads them once: 32 sequences of 16000 slots (262 MB), 64 heads over 1, 260 MB and 96 us, by
// the order alone, on four dies, 1026 MB and 153; 32 over 1 61 and 81.
constexpr int kWaves = 4;
struct PagedPiece {
    int b, unit, piece, n, q;  // piece number `piece` of n, q tiles each; n = 0: none
    int more;                  // the place of the unit's second piece (for a first piece: where B <= 64)
    int span;                  // paged_span of sequence b
};
// The place of workgroup w: of 8 `tiles` places in a row, number 8 t + x takes the one of tile t of the x-th keys.
__device__ __forceinline__ int paged_place(const PagedAttn& a, int w) {
    if (a.tiles == 1) return w;
    const int run = 8 * a.tiles, in = w % run;
    return w - in + run > a.groups ? w : w - in + in % 8 * a.tiles + in / 8;
}
// The place of piece s of unit u of the launch.
__device__ __forceinline__ int paged_group(int s, int u, int more, int tiles) { return s ? more + (s - 1) * tiles : u; }

template <bool STEP, int TK>
__device__ __forceinline__ PagedPiece paged_piece(const PagedAttn& a, int w, int lane) {
    const int B = a.c.B, per = a.c.Hkv * a.tiles, units = B * per, room = a.groups - units;
    PagedPiece p{};
    if (room == 0) {
        p.b = w / per;
        p.unit = w - p.b * per;
        p.n = 1;
        p.q = INT_MAX / 2;
        p.span = paged_span<STEP>(a, a.c.lens[p.b]);
        return p;
    }
    int span = 0;
    auto tiles = [&](int b) {
        span = b < B ? paged_span<STEP>(a, a.c.lens[b]) : 0;
        return (span + TK - 1) / TK;
    };
    // ceil(nb / q), 1 at least: nb <= 2^16, and 1 / q is good to 2^-23, so the quarter decides
    auto pieces = [&](int nb, int q) { return nb <= q ? 1 : (int)(((float)(nb + q - 1) + 0.25f) * __builtin_amdgcn_rcpf((float)q)); };
    const int mine = tiles(lane);
    int q, n = 1, incl = 0;  // incl: pieces past the first of this lane's sequence and those before it
    if (B <= 64) {
        const float all = (float)__builtin_amdgcn_readlane(paged_scan(mine), 63);
        // (the last pieces are half empty on the average)
        q = max(kWaves, (int)(all * (float)per * __builtin_amdgcn_rcpf((float)room + 0.6f * (float)units)));
        for (;; q += max(1, q / 32)) {  // (ends at the latest when q tiles are the longest sequence)
            n = pieces(mine, q);
            incl = paged_scan(n - 1);
            if (__builtin_amdgcn_readlane(incl, 63) * per <= room) break;
        }
    } else {  // all / q pieces past the first ones at most: q from that
        int all = mine, most = mine;
        for (int b = 64; b < B; b += 64) {
            const int nb = tiles(b + lane);
            all += nb;
            most = max(most, nb);
        }
        all = __builtin_amdgcn_readlane(paged_scan(all), 63);
        most = lane63(wave_reduce63(most, 0, [](int x, int y) { return max(x, y); }));
        q = max(kWaves, (int)fminf((float)all * (float)per / (float)room * 1.0001f, 1e6f) + 1);
        if (w >= units && most <= q) return p;
    }
    if (w < units) {
        p.b = w / per;
        p.unit = w - p.b * per;
        if (B <= 64) {
            p.n = __builtin_amdgcn_readlane(n, p.b);
            p.span = __builtin_amdgcn_readlane(span, p.b);
            const int ht = a.tiles == 1 ? 0 : p.unit % a.tiles;
            p.more = units + (__builtin_amdgcn_readlane(incl, p.b) - p.n + 1) * per + (p.unit - ht) * (p.n - 1) + ht;
        } else {
            p.span = paged_span<STEP>(a, a.c.lens[p.b]);
            p.n = pieces((p.span + TK - 1) / TK, q);
        }
    } else {
        const int e = w - units;
        int at = 0, before = 0;
        unsigned long long here = 0ull;
        for (;; at += 64) {
            if (at >= B) return p;
            if (B > 64) {
                n = pieces(tiles(at + lane), q);
                incl = paged_scan(n - 1) + before;
                before = __builtin_amdgcn_readlane(incl, 63);
            }
            here = __ballot(e < incl * per);
            if (here != 0ull) break;
        }
        const int l = (int)__builtin_ctzll(here), others = __builtin_amdgcn_readlane(n, l) - 1;
        const int start = (__builtin_amdgcn_readlane(incl, l) - others) * per;
        p.b = at + l;
        p.n = others + 1;
        p.span = __builtin_amdgcn_readlane(span, l);
        const int kh = (e - start) / (others * a.tiles), in = e - start - kh * others * a.tiles, s = a.tiles == 1 ? in : in / a.tiles;
        const int ht = in - s * a.tiles;
        p.unit = kh * a.tiles + ht;
        p.piece = 1 + s;
        p.more = units + start + kh * others * a.tiles + ht;
    }
    p.q = ((p.span + TK - 1) / TK + p.n - 1) / p.n;
    return p;
}

// A unit's pieces are joined by the workgroup that ends last, where they are few (paged_shape).  Which one that is, its ticket
// tells: a word of the launch's nonce and a count.  The workspace needs no clearing: the nonce is a number that none of the last
// 2^44 launches of the process has had, a word of another is set to (nonce, 0) by whoever finds it so (if that fails, another has done it),
// and the last leaves 0, so that the same launch can be replayed.  Sums go from one workgroup to the other past the caches of
// their dies: stored and loaded coherent with the device, the stores done (s_waitcnt) before the count.
constexpr int kTicketBits = 20;

__device__ __forceinline__ void paged_put(float* at, float x, float y) {
    __hip_atomic_store(reinterpret_cast<unsigned long long*>(at),
                       (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ v2f paged_get(const float* at) {
    const unsigned long long w =
        __hip_atomic_load(reinterpret_cast<const unsigned long long*>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return v2f{__uint_as_float((unsigned)w), __uint_as_float((unsigned)(w >> 32))};
}
// Whether slots s .. s + 3 (s % 4 == 0, so of one page) are there: weights of those in a hole are left alone, where a head
// whose sum is NaN would leave a NaN.
__device__ __forceinline__ bool paged_there(const PagedCache& c, int b, int s) {
    const int id = c.table[(size_t)b * c.P + (s >> c.shift)];
    return id >= 0 && id < c.pages;
}
// What the slots of unit u weighed, by the workgroup that has its heads' totals ((reference, 1 / sum of weights) a row): scores, as
// all workgroups of the unit have stored them, to the KV head's accumulated weights.
__device__ __forceinline__ void paged_weigh(const PagedAttn& a, const float* score, int bk, int len, int rows, int TK, const float (*total)[2],
                                            int t) {
    for (int s0 = t * 4; s0 < len; s0 += 256 * kWaves) {
        const float* const at = score + s0 / TK * rows * TK + s0 % TK;
        float* const w = a.weights + (size_t)bk * a.slots + s0;
        const bool there = paged_there(a.c, bk / a.c.Hkv, s0);
        v4f add{};
#pragma unroll 8
        for (int row = 0; row < rows; ++row) {
            const v2f lo = paged_get(at + row * TK), hi = paged_get(at + row * TK + 2);
            const float ref = total[row][0], inv = total[row][1];
            add += v4f{__builtin_amdgcn_exp2f(lo[0] - ref), __builtin_amdgcn_exp2f(lo[1] - ref), __builtin_amdgcn_exp2f(hi[0] - ref),
                       __builtin_amdgcn_exp2f(hi[1] - ref)} * inv;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (there && s0 + e < len) w[e] += add[e];
    }
}
// True for the workgroup that joined.  room: LDS for kLastMost floats and, behind them, a row's sums a group of threads; flag: a word
// of LDS; total: its rows'.
constexpr int kLastMost = 64;  // pieces times heads that the last workgroup joins
template <int HD>
__device__ __forceinline__ bool paged_last(const PagedAttn& a, const PagedPiece& p, int u, unsigned long long* ticket, float* out, int rows,
                                           float* room, int* flag, float (*total)[2], int t, int lane, int wave) {
    constexpr int L = HD / 4, NT = 64 * kWaves;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t == 0) {
        const unsigned long long c = __hip_atomic_fetch_add(ticket, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool last = (int)(c & ((1u << kTicketBits) - 1)) + 1 == p.n;
        if (last) __hip_atomic_store(ticket, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = last;
    }
    __syncthreads();
    if (!*flag) return false;
    auto part = [&](int s, int e) { return a.part + (size_t)paged_group(s, u, p.more, a.tiles) * 16 * HD + e * 4; };
    const int n = p.n, cols = rows * L, groups = max(NT / cols, 1), grp = t / cols;
    float* const factor = room;  // [rows][n]
    v4f* const sums = reinterpret_cast<v4f*>(room + kLastMost);
    constexpr int kAhead = 8;
    v2f ahead[kAhead][2];
    auto load = [&](int e) {  // of a group's first pieces
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int s = grp + k * groups;
            if (s < n) {
                ahead[k][0] = paged_get(part(s, e));
                ahead[k][1] = paged_get(part(s, e) + 2);
            }
        }
    };
    int e = t - grp * cols;
    const bool mine = grp < groups && e < cols;
    if (mine) load(e);  // (while the references come)
    for (int row = wave; row < rows; row += kWaves) {
        const v2f x = lane < n ? paged_get(a.ml + (size_t)paged_group(lane, u, p.more, a.tiles) * 32 + row * 2) : v2f{-INFINITY, 0.0f};
        const float top = lane63(wave_reduce63(x[0], -INFINITY, [](float x, float y) { return fmaxf(x, y); }));
        const float ref = top > -INFINITY ? top : 0.0f, f = __builtin_amdgcn_exp2f(x[0] - ref);
        const float sum = lane63(wave_reduce63(x[1] * f, 0.0f, [](float x, float y) { return x + y; }));
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;  // (no slot: zeros)
        if (lane < n) factor[row * n + lane] = f * inv;
        if (lane == 0) {
            total[row][0] = ref;
            total[row][1] = inv;
        }
    }
    __syncthreads();
    for (; mine && e < cols; e += NT) {  // (one round where there are several groups)
        const float* const weight = factor + e / L * n;
        v4f y{};
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int s = grp + k * groups;
            if (s < n) y += v4f{ahead[k][0][0], ahead[k][0][1], ahead[k][1][0], ahead[k][1][1]} * weight[s];
        }
        for (int s = grp + kAhead * groups; s < n; s += groups) {
            const v2f lo = paged_get(part(s, e)), hi = paged_get(part(s, e) + 2);
            y += v4f{lo[0], lo[1], hi[0], hi[1]} * weight[s];
        }
        if (groups > 1) sums[t] = y;
        else *reinterpret_cast<v4f*>(out + e * 4) = y;
        if (e + NT < cols) load(e + NT);
    }
    if (groups == 1) return true;
    __syncthreads();
    if (t < cols) {
        v4f y = sums[t];
        for (int w = 1; w < groups; ++w) y += sums[w * cols + t];
        *reinterpret_cast<v4f*>(out + t * 4) = y;
    }
    return true;
}

template <int T, int HD, bool STEP, bool ONCE>
__global__ void __launch_bounds__(64 * kWaves, 2) paged_attn_kernel(PagedAttn a) {
    typedef AttnTile<T, HD, ONCE> Tile;
    typedef typename Tile::E E;
    constexpr int TK = Tile::TK, L = HD / 4;
    // the queries, and in their place, when all waves have taken them, the waves' sums
    constexpr int kPart = kWaves * 16 * (HD + 4) * 4;
    __shared__ __align__(16) char both[kPart > Tile::QBYTES ? kPart : Tile::QBYTES];
    __shared__ float ml[kWaves][16][2];
    __shared__ int power[16];
    __shared__ float total[16][2];
    __shared__ __align__(16) E fresh[2][STEP ? HD : 16];
    float(*const part)[16][HD + 4] = reinterpret_cast<float(*)[16][HD + 4]>(both);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), i = lane & 15, g = lane >> 4;
    const int place = paged_place(a, blockIdx.x);
    const PagedPiece p = paged_piece<STEP, TK>(a, place, lane);
    if (p.n == 0) return;
    const int b = p.b, kh = p.unit / a.tiles, ht = p.unit - kh * a.tiles, bk = b * a.c.Hkv + kh, u = b * a.c.Hkv * a.tiles + p.unit;
    const int len = p.span, tiles = (len + TK - 1) / TK, first = min(p.piece * p.q, tiles);
    int last = min(first + p.q, tiles);
    const int newest = STEP ? paged_newest(a, b, len) : 0;
    const int rows = min(a.G - 16 * ht, 16);
    const int h0 = kh * a.G + 16 * ht;  // the tile's first head
    float* const score = a.scores ? a.scores + ((size_t)b * a.H + h0) * paged_even(a.c.P << a.c.shift) : nullptr;  // the unit's
    // the unit's ticket: whatever the memory held, the first to come makes it this launch's, with none counted
    unsigned long long* const ticket = a.whole && p.n > 1 ? a.tickets + u : nullptr;
    unsigned long long held = 0ull;
    if (ticket && t == 0) held = __hip_atomic_load(ticket, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    auto claim = [&] {
        if (ticket && t == 0 && held >> kTicketBits != a.nonce)
            __hip_atomic_compare_exchange_strong(ticket, &held, a.nonce << kTicketBits, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT);
    };
    Tile x;
    float m = -INFINITY, l = 0.0f;
    x.clear();
    if (first >= last) claim();
    else {
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
        int at = first + wave, n = 0;
        bool there0 = false, there1 = false, next0 = false, next1 = false;
        const E *b0 = kbase, *b1 = kbase;
        if (at < last) {
            look(at);
            b0 = base(n, at, 0, there0);
            b1 = TK == 32 ? base(n, at, 1, there1) : b0;
            x.load_k(b0, b1, i, g);
            x.load_v(b0 + a.c.kv_stride, b1 + a.c.kv_stride, i, g);
        }
        // the queries, rotated where the step asks for it, into LDS; a step's new row too, where this piece has the last tile
        if (newest < 0) last = at = first;  // (a step without a place: nothing from here on)
        const float* const cs = STEP && newest >= 0 ? a.n.rope + (size_t)a.n.pos[b] * a.n.rotary : nullptr;
        const int items = newest < 0 ? 0 : rows * L, more = STEP && last == tiles ? 2 * L : 0;
        for (int e = t; e < items + more; e += 64 * kWaves) {
            const int d = e % L * 4, row = e / L;
            if (row < rows) {
                const float* const src = a.q + ((size_t)b * a.H + h0 + row) * HD;
                const v4f y = STEP ? paged_rotate4(src, cs, d, a.n.rotary, a.n.interleaved) : *reinterpret_cast<const v4f*>(src + d);
                int pw = 0;
                if constexpr (Tile::F16) {  // the head's largest into [2^14, 2^15): over the L lanes that have it
                    float big = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
#pragma unroll
                    for (int w = 1; w < L; w <<= 1) big = fmaxf(big, __shfl_xor(big, w, 64));
                    pw = min(max(14 + 127 - (int)(__float_as_uint(big) >> 23), -113), 120);
                    if (d == 0) power[row] = pw;
                }
                Tile::stage(both, y, row, d, pw);
            } else if constexpr (STEP) {
                const bool is_v = row > rows;
                const float* const src = (is_v ? a.n.v : a.n.k) + (size_t)bk * HD;
                const v4f y = is_v ? *reinterpret_cast<const v4f*>(src + d) : paged_rotate4(src, cs, d, a.n.rotary, a.n.interleaved);
                paged_store4<T>(&fresh[is_v][d], y);
                if (ht == 0)
                    paged_store4<T>(const_cast<E*>(kbase) + (is_v ? a.c.kv_stride : 0) + (long long)newest * a.c.page_stride +
                                        ((len - 1) & in_page) * HD + d, y);
            }
        }
        __syncthreads();
        claim();
        x.take(both, Tile::F16 ? power[min(i, rows - 1)] : 0, a.scale, min(i, rows - 1), g);  // (columns past the last head repeat it)
        for (; at < last; at += kWaves, ++n, there0 = next0, there1 = next1) {
            const bool more = at + kWaves < last;
            if constexpr (STEP)
                if (at == tiles - 1) x.put(fresh[0], fresh[1], len - 1 - at * TK, i, g);
            float s[Tile::NS];
            x.scores(s);
            if (more) {
                if (((n + 1) & 63) == 0) look(at + kWaves);
                b0 = base(n + 1, at + kWaves, 0, next0);
                b1 = TK == 32 ? base(n + 1, at + kWaves, 1, next1) : b0;
                x.load_k(b0, b1, i, g);
            }
            if (at == tiles - 1 || !there0 || (TK == 32 && !there1)) {
#pragma unroll
                for (int e = 0; e < Tile::NS; ++e) {
                    if (at * TK + Tile::slot(e, g) >= len || !(TK == 32 && e >= 4 ? there1 : there0)) {
                        s[e] = -INFINITY;
                        x.hide(e);
                    }
                }
            }
            float raw[Tile::NS];
#pragma unroll
            for (int e = 0; e < Tile::NS; ++e) raw[e] = s[e];
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
            if (score && i < rows) {  // (behind the loads: a wave waits for its accesses in their order)
                float* const to = score + (at * rows + i) * TK;
#pragma unroll
                for (int e = 0; e < Tile::NS; e += 4) {
                    if (a.whole) {
                        paged_put(to + Tile::slot(e, g), raw[e], raw[e + 1]);
                        paged_put(to + Tile::slot(e, g) + 2, raw[e + 2], raw[e + 3]);
                    } else *reinterpret_cast<v4f*>(to + Tile::slot(e, g)) = v4f{raw[e], raw[e + 1], raw[e + 2], raw[e + 3]};
                }
            }
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
    for (int e = t; e < rows * L; e += 64 * kWaves) {
        const int row = e / L, d = e % L * 4;
        v4f y = *reinterpret_cast<const v4f*>(&part[0][row][d]);
#pragma unroll
        for (int w = 1; w < kWaves; ++w) y += *reinterpret_cast<const v4f*>(&part[w][row][d]);
        float top = ml[0][row][0], sum = 0.0f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, ml[w][row][0]);
        const float at = top > -INFINITY ? top : 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += ml[w][row][1] * __builtin_amdgcn_exp2f(ml[w][row][0] - at);
        if (p.n == 1) {
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;  // (no slot: zeros)
            *reinterpret_cast<v4f*>(a.out + ((size_t)b * a.H + h0 + row) * HD + d) = y * inv;
            if (d == 0) {
                total[row][0] = at;
                total[row][1] = inv;
            }
        } else if (a.whole) {
            paged_put(a.part + ((size_t)place * 16 + row) * HD + d, y[0], y[1]);
            paged_put(a.part + ((size_t)place * 16 + row) * HD + d + 2, y[2], y[3]);
            if (d == 0) paged_put(a.ml + ((size_t)place * 16 + row) * 2, top, sum);
            continue;
        } else *reinterpret_cast<v4f*>(a.part + ((size_t)place * 16 + row) * HD + d) = y;
        if (d == 0 && a.ml) *reinterpret_cast<v2f*>(a.ml + ((size_t)place * 16 + row) * 2) = v2f{top, sum};
    }
    if (a.whole) {
        bool mine = true;
        if (p.n > 1)
            mine = paged_last<HD>(a, p, u, ticket, a.out + ((size_t)b * a.H + h0) * HD, rows, reinterpret_cast<float*>(both), power, total, t,
                                  lane, wave);
        if (!mine || !score || newest < 0) return;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        paged_weigh(a, score, bk, len, rows, TK, total, t);
        return;
    }
    if (t == 0 && a.ml && p.piece == (p.n > 1)) a.units[u] = make_int2(p.more, p.n);
}

// Head number `row` of unit u: its reference (the largest of its pieces') and the reciprocal of its sum of weights, found by a
// wave; unit: the place of its second piece, and how many pieces there are.
__device__ __forceinline__ void paged_total(const PagedAttn& a, int u, int2 unit, int row, int lane, float& ref, float& inv) {
    auto ml = [&](int s) { return a.ml + (size_t)paged_group(s, u, unit.x, a.tiles) * 32 + row * 2; };
    const int n = unit.y;
    float top = -INFINITY;
    for (int s = lane; s < n; s += 64) top = fmaxf(top, ml(s)[0]);
    top = lane63(wave_reduce63(top, -INFINITY, [](float x, float y) { return fmaxf(x, y); }));
    ref = top > -INFINITY ? top : 0.0f;
    float sum = 0.0f;
    for (int s = lane; s < n; s += 64) sum += ml(s)[1] * __builtin_amdgcn_exp2f(ml(s)[0] - ref);
    sum = lane63(wave_reduce63(sum, 0.0f, [](float x, float y) { return x + y; }));
    inv = sum != 0.0f ? 1.0f / sum : 0.0f;  // (no slot: zeros)
}

// The join: workgroups [0, B H): a head's pieces into its output; the others: what 4 NT slots of a KV head weighed (every
// head's score against its reference and sum), added to the accumulated weights.
constexpr int kJoinHeads = 1024;  // H / Hkv at most

template <int HD, bool STEP, int NT>
__global__ void __launch_bounds__(NT) paged_join_kernel(PagedAttn a, int TK, int joins, int chunks) {
    constexpr int L = HD / 4;
    __shared__ float sums[NT / L][HD];
    __shared__ float total[kJoinHeads][2];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    if ((int)blockIdx.x < joins) {
        const int head = blockIdx.x % a.H, b = blockIdx.x / a.H, kh = head / a.G, in = head % a.G;
        const int u = (b * a.c.Hkv + kh) * a.tiles + in / 16;
        const int2 unit = a.units[u];
        const int n = unit.y;
        if (n == 1) return;
        const int d = t % L * 4, grp = t / L;
        auto place = [&](int s) { return (size_t)paged_group(s, u, unit.x, a.tiles) * 16 + in % 16; };
        auto part = [&](int s) { return *reinterpret_cast<const v4f*>(a.part + place(s) * HD + d); };
        v4f y{};
        float own = -INFINITY, ref, inv;
        if (grp < n) {  // (before the references are known, which takes as long as these loads)
            y = part(grp);
            own = a.ml[place(grp) * 2];
        }
        paged_total(a, u, unit, in % 16, lane, ref, inv);
        y *= __builtin_amdgcn_exp2f(own - ref);
#pragma unroll 4
        for (int s = grp + NT / L; s < n; s += NT / L) y += part(s) * __builtin_amdgcn_exp2f(a.ml[place(s) * 2] - ref);
        *reinterpret_cast<v4f*>(&sums[grp][d]) = y;
        __syncthreads();
        if (grp) return;
#pragma unroll
        for (int w = 1; w < NT / L; ++w) y += *reinterpret_cast<const v4f*>(&sums[w][d]);
        *reinterpret_cast<v4f*>(a.out + ((size_t)b * a.H + head) * HD + d) = y * inv;
        return;
    }
    const int chunk = ((int)blockIdx.x - joins) % chunks, bk = ((int)blockIdx.x - joins) / chunks, b = bk / a.c.Hkv, kh = bk % a.c.Hkv;
    const int len = paged_span<STEP>(a, a.c.lens[b]), cap = a.c.P << a.c.shift, s0 = (chunk * NT + t) * 4;
    if (chunk * NT * 4 >= len || (STEP && paged_newest(a, b, len) < 0)) return;
    for (int in = wave; in < a.G; in += NT / 64) {
        float ref, inv;
        const int u = bk * a.tiles + in / 16;
        paged_total(a, u, a.units[u], in % 16, lane, ref, inv);
        total[in][0] = ref;
        total[in][1] = inv;
    }
    __syncthreads();
    if (s0 >= len) return;
    const bool there = paged_there(a.c, b, s0);
    v4f add{};
    for (int h = 0; h < a.G; h += 16) {
        const int rows = min(a.G - h, 16);
        const float* const score = a.scores + ((size_t)b * a.H + kh * a.G + h) * paged_even(cap) + s0 / TK * rows * TK + s0 % TK;
#pragma unroll 4
        for (int in = 0; in < rows; ++in) {
            const v4f s = *reinterpret_cast<const v4f*>(score + in * TK);
#pragma unroll
            for (int e = 0; e < 4; ++e) add[e] += __builtin_amdgcn_exp2f(s[e] - total[h + in][0]) * total[h + in][1];
        }
    }
    float* const w = a.weights + (size_t)bk * a.slots + s0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (there && s0 + e < len) w[e] += add[e];
}

// ---- eviction ----------------------------------------------------------------------------
// Which slots are kept: the last `recent`, and of those before them (the judged) the largest weights, ties to the lowest slot;
// slots in holes are not there.  Weights are taken as whole numbers of the same order (NaN above all, -0 as 0; 0 for what is not
// there).  The smallest that is kept is found from histograms of its upper 11 bits, of the next 11 among those that have these,
// and of the last 10.  Then every wave counts the kept of its run of slots, and writes them out behind those of the waves before.
// A workgroup of 1024 threads takes a KV head of a sequence, up to 32 slots a thread, in registers (of 17 to 32 a part spills: 28
// registers, 116 bytes a lane; 16000 slots cut to half, 5 heads of 128, 25 us, 24000 41); longer caches are shared among
// workgroups of 8 slots a thread, in a launch for every histogram and two for the output, all launches us, alone / shared: 5 heads
// of 16000 slots 16 / 32, 32000 33 / 32 (and five launches more on the host), 80 heads 39 / 49, 300 heads 69 / 99; 10 heads of
// 131072 slots by one workgroup each, the weights read again for every pass, 359 / 35.  Bound by the passes' latencies: 128 heads of up
// to 8191 slots take 12 us for 12 MB.
constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64, kEvictBins = 2048;
constexpr int kEvictAlone = 32 * kEvictThreads, kEvictChunk = 8 * kEvictThreads;

__device__ __forceinline__ unsigned evict_key(float w) {  // 1 and up (0: not there)
    unsigned u = __float_as_uint(w);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
    if (u == 0x80000000u) u = 0u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ int evict_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ int evict_bins(int pass) { return pass == 2 ? 1024 : 2048; }

// A head's slots in a workgroup: `run` a wave from s0 on, thread by thread, R a thread at most.  key[j], mine and there of slot
// s0 + 64 j + lane: keys of the judged, 0 for others; stay: bit j, a recent slot that is there.
template <int R>
struct EvictSlots {
    unsigned key[R], stay;
    int s0, n;
    __device__ __forceinline__ void load(const PagedEvict& a, int bk, int from, int to, int len, int lane, int wave) {
        n = (to - from + kEvictThreads - 1) / kEvictThreads;
        s0 = from + wave * 64 * n;
        const int b = bk / a.c.Hkv, old = max(len - a.recent, 0);
        const int* const row = a.c.table + (size_t)b * a.c.P;
        const float* const w = a.weights + (size_t)bk * a.slots;
        stay = 0u;
        int id[R];
        float x[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int s = s0 + 64 * j + lane;
            const bool in = j < n && s < to;
            id[j] = in ? row[s >> a.c.shift] : -1;
            x[j] = in && s < old ? w[s] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int s = s0 + 64 * j + lane;
            const bool there = id[j] >= 0 && id[j] < a.c.pages;
            key[j] = there && s < old ? evict_key(x[j]) : 0u;
            if (there && s >= old) stay |= 1u << j;
        }
    }
    // one histogram in LDS (bins cleared before; a barrier behind): of the keys with `prefix` under `mask`
    __device__ __forceinline__ void count(int* hist, int pass, unsigned prefix, unsigned mask) const {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const unsigned k = key[j];
            if (j < n && k && (k & mask) == prefix) atomicAdd(&hist[(k >> evict_shift(pass)) & (evict_bins(pass) - 1)], 1);
        }
    }
    // how many lie above `prefix` (or stay), and how many are equal to it: of this wave, in every lane
    __device__ __forceinline__ void sums(unsigned prefix, int& above, int& equal) const {
        above = __popc(stay);
        equal = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            above += key[j] > prefix ? 1 : 0;
            equal += key[j] && key[j] == prefix ? 1 : 0;
        }
        above = __builtin_amdgcn_readlane(paged_scan(above), 63);
        equal = __builtin_amdgcn_readlane(paged_scan(equal), 63);
    }
    // the kept ones number lo .. hi - 1, out: kept before this wave's; equal: equal ones before it, of which the first `want` are
    // kept; list: their slots in LDS too
    __device__ __forceinline__ void write(const PagedEvict& a, int bk, unsigned prefix, int want, int out, int equal, int lane, int lo, int hi,
                                          int* list) const {
        int* const kept = a.kept + (size_t)bk * a.keep;
        float* const left = a.new_weights + (size_t)bk * a.slots;
        const float* const w = a.weights + (size_t)bk * a.slots;
        const unsigned long long below = (1ull << lane) - 1;
        constexpr int N = R < 8 ? R : 8;
#pragma unroll
        for (int j0 = 0; j0 < R; j0 += N) {
            if (j0 >= n) break;
            float x[N];  // (asked for at once, not one by one behind each slot's decision)
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = key[j0 + j] || (stay >> (j0 + j) & 1u) ? w[s0 + 64 * (j0 + j) + lane] : 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const unsigned k = key[j0 + j];
                const bool same = k && k == prefix;
                const unsigned long long e = __ballot(same);
                const bool keep = (stay >> (j0 + j) & 1u) || k > prefix || (same && equal + __popcll(e & below) < want);
                const unsigned long long all = __ballot(keep);
                const int at = out + __popcll(all & below);
                if (keep && at >= lo && at < hi) {
                    kept[at] = s0 + 64 * (j0 + j) + lane;
                    left[at] = x[j];
                    if (list) list[at - lo] = s0 + 64 * (j0 + j) + lane;
                }
                equal += __popcll(e);
                out += __popcll(all);
            }
        }
    }
};

// From a histogram: the bin that the key of number `want`, counted from the largest, is in, and its number there.  True where the
// whole bin is kept.
__device__ __forceinline__ bool evict_find(const int* hist, int pass, int (*totals)[2], int* found, unsigned& prefix, unsigned& mask,
                                           int& want, int t, int lane, int wave) {
    const int bins = evict_bins(pass), hi = bins - 1 - 2 * t;  // from the largest bin down, two a thread
    const int n0 = hi >= 0 ? hist[hi] : 0, n1 = hi >= 1 ? hist[hi - 1] : 0, incl = paged_scan(n0 + n1);
    if (lane == 63) totals[wave][0] = incl;
    __syncthreads();
    int before = incl - n0 - n1;
#pragma unroll
    for (int v = 0; v < kEvictWaves; ++v) before += v < wave ? totals[v][0] : 0;
    if (n0 && before < want && before + n0 >= want) {
        found[0] = hi;
        found[1] = want - before;
        found[2] = n0;
    } else if (n1 && before + n0 < want && before + n0 + n1 >= want) {
        found[0] = hi - 1;
        found[1] = want - before - n0;
        found[2] = n1;
    }
    __syncthreads();
    prefix |= (unsigned)found[0] << evict_shift(pass);
    mask |= (unsigned)(bins - 1) << evict_shift(pass);
    want = found[1];
    return want == found[2];
}

// What is left of a head's outputs behind its last kept slot, by `threads` threads.
__device__ __forceinline__ void evict_rest(const PagedEvict& a, int bk, int total, int t, int threads) {
    int* const kept = a.kept + (size_t)bk * a.keep;
    float* const left = a.new_weights + (size_t)bk * a.slots;
    for (int n = total + t; n < a.keep; n += threads) kept[n] = -1;
    for (int n = total + t; n < a.slots; n += threads) left[n] = 0.0f;
    if (bk % a.c.Hkv == 0 && t == 0) a.new_lens[bk / a.c.Hkv] = total;  // (the same for every head: holes are the sequence's)
}

// A kept slot's row of K and of V into the new table's page, 16 bytes a thread, past the caches (16 sequences of 1000 to 8191 cut
// to 4096: the whole eviction 63.4 us through them, so 59.8).  n: its number; o: the thread's bytes of the row.
__device__ __forceinline__ void evict_move(const PagedEvict& a, int b, int kh, int s, int n, int o, int row_bytes, int esize) {
    const int in_page = (1 << a.c.shift) - 1;
    const int from = a.c.table[(size_t)b * a.c.P + (s >> a.c.shift)], to = a.new_table[(size_t)b * a.new_P + (n >> a.c.shift)];
    if (from < 0 || from >= a.c.pages || to < 0 || to >= a.c.pages) return;
    char* const base = static_cast<char*>(a.c.cache) + ((long long)kh << a.c.shift) * row_bytes + o;
    const long long src = (long long)from * a.c.page_stride * esize + (long long)(s & in_page) * row_bytes;
    const long long dst = (long long)to * a.c.page_stride * esize + (long long)(n & in_page) * row_bytes;
    const long long v = a.c.kv_stride * esize;
    const v4u x = paged_load<true, v4u>(base + src), y = paged_load<true, v4u>(base + src + v);
    __builtin_nontemporal_store(x, reinterpret_cast<v4u*>(base + dst));
    __builtin_nontemporal_store(y, reinterpret_cast<v4u*>(base + dst + v));
}

// The whole of it, for a share of a head's kept slots: every workgroup of a head makes the same selection, and each moves
// its own `share` rows, so that one launch does both: a chat's 2048 slots cut to 1024 15.0 us in two launches, so 12.6; 16
// sequences of up to 8191 cut to 4096 58.4 / 58.5 on the GPU.
constexpr int kEvictShare = 4096;
template <int R>
__global__ void __launch_bounds__(kEvictThreads) paged_select_kernel(PagedEvict a, int parts, int share, int row_bytes, int esize) {
    __shared__ int hist[kEvictBins];
    __shared__ int totals[kEvictWaves][2], found[3];
    __shared__ int list[kEvictShare];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int part = blockIdx.x % parts, bk = blockIdx.x / parts, b = bk / a.c.Hkv, lo = part * share;
    const int len = min(max(a.c.lens[bk / a.c.Hkv], 0), a.c.P << a.c.shift);
    EvictSlots<R> x;
    x.load(a, bk, 0, len, len, lane, wave);
    hist[t] = hist[t + kEvictThreads] = 0;
    int stay, judged;
    x.sums(0u, stay, judged);  // (every judged one lies above 0)
    judged = stay - __builtin_amdgcn_readlane(paged_scan(__popc(x.stay)), 63);
    if (lane == 0) {
        totals[wave][0] = stay - judged;
        totals[wave][1] = judged;
    }
    __syncthreads();
    stay = judged = 0;
#pragma unroll
    for (int v = 0; v < kEvictWaves; ++v) {
        stay += totals[v][0];
        judged += totals[v][1];
    }
    int want = min(judged, a.keep - stay);  // of the judged ones (recent <= keep)
    unsigned prefix = 0u, mask = 0u;
    if (want > 0 && want < judged) {
        for (int pass = 0; pass < 3; ++pass) {
            if (pass) {
                hist[t] = hist[t + kEvictThreads] = 0;
                __syncthreads();
            }
            x.count(hist, pass, prefix, mask);
            __syncthreads();
            if (evict_find(hist, pass, totals, found, prefix, mask, want, t, lane, wave)) {
                prefix = max(prefix, 1u) - 1u;  // right below the bin (keys are 1 and up), and none of those equal to it
                want = 0;
                break;
            }
        }
    } else {  // all of them, or none
        prefix = want > 0 ? 0u : 0xFFFFFFFFu;
        want = 0;
    }
    int above, equal;
    x.sums(prefix, above, equal);
    __syncthreads();
    if (lane == 0) {
        totals[wave][0] = above;
        totals[wave][1] = equal;
    }
    __syncthreads();
    int before = 0, same = 0, all = 0, equals = 0;
#pragma unroll
    for (int v = 0; v < kEvictWaves; ++v) {
        before += v < wave ? totals[v][0] : 0;
        same += v < wave ? totals[v][1] : 0;
        all += totals[v][0];
        equals += totals[v][1];
    }
    const int total = all + min(equals, want), hi = min(lo + share, total);
    x.write(a, bk, prefix, want, before + min(same, want), same, lane, lo, hi, list);
    evict_rest(a, bk, total, part * kEvictThreads + t, parts * kEvictThreads);
    __syncthreads();
    const int lanes = row_bytes / 16;
#pragma unroll 4
    for (int n = lo + t / lanes; n < hi; n += kEvictThreads / lanes)
        evict_move(a, b, bk - b * a.c.Hkv, list[n - lo], n, t % lanes * 16, row_bytes, esize);
}

// The same in several launches (step 0 to 4), workgroup (head, chunk of kEvictChunk slots): histograms 0 to 2, the chunks' counts, the
// output.  work, a head: [0] stay, [1] judged, [2 ..] histograms, then a word pair (prefix, want) a step, then (above, equal) a chunk.
constexpr int kEvictState = 2 + 3 * kEvictBins, kEvictWords = kEvictState + 2 * 3;

__global__ void __launch_bounds__(kEvictThreads) paged_clear_kernel(int* work, int words) {
    for (int n = threadIdx.x; n < kEvictState; n += kEvictThreads) work[(size_t)blockIdx.x * words + n] = 0;
}
template <int STEP>
__global__ void __launch_bounds__(kEvictThreads) paged_share_kernel(PagedEvict a, int* work, int words, int chunks) {
    __shared__ int hist[STEP < 3 ? kEvictBins : 1];
    __shared__ int totals[kEvictWaves][2], found[3];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int chunk = blockIdx.x % chunks, bk = blockIdx.x / chunks;
    const int len = min(max(a.c.lens[bk / a.c.Hkv], 0), a.c.P << a.c.shift), from = chunk * kEvictChunk;
    int* const own = work + (size_t)bk * words;
    int* const counts = own + kEvictWords;
    // (a chunk behind the slots still says that it has none, and step 4's clears)
    EvictSlots<8> x;
    x.load(a, bk, from, max(from, min(from + kEvictChunk, len)), len, lane, wave);
    if constexpr (STEP == 0) {
        hist[t] = hist[t + kEvictThreads] = 0;
        __syncthreads();
        x.count(hist, 0, 0u, 0u);
        int above, equal;
        x.sums(0u, above, equal);
        const int stay = __builtin_amdgcn_readlane(paged_scan(__popc(x.stay)), 63);
        if (lane == 0) {
            if (stay) atomicAdd(&own[0], stay);
            if (above - stay) atomicAdd(&own[1], above - stay);
        }
        __syncthreads();
        for (int n = t; n < kEvictBins; n += kEvictThreads)
            if (hist[n]) atomicAdd(&own[2 + n], hist[n]);
        return;
    }
    // what the step before has found
    const int stay = own[0], judged = own[1];
    unsigned prefix = 0u, mask = 0u;
    int want = min(judged, a.keep - stay);
    const bool search = want > 0 && want < judged;
    if (!search) {
        prefix = want > 0 ? 0u : 0xFFFFFFFFu;
        want = 0;
    } else if (STEP < 4) {
        if (STEP > 1) {
            prefix = (unsigned)own[kEvictState + 2 * (STEP - 2)];
            want = own[kEvictState + 2 * (STEP - 2) + 1];
            mask = STEP == 2 ? 0xFFE00000u : 0xFFFFFC00u;
        }
        evict_find(own + 2 + (STEP - 1) * kEvictBins, STEP - 1, totals, found, prefix, mask, want, t, lane, wave);
        if (chunk == 0 && t == 0) {
            own[kEvictState + 2 * (STEP - 1)] = (int)prefix;
            own[kEvictState + 2 * (STEP - 1) + 1] = want;
        }
    } else {
        prefix = (unsigned)own[kEvictState + 4];
        want = own[kEvictState + 5];
    }
    if constexpr (STEP < 3) {
        if (!search) return;
        hist[t] = hist[t + kEvictThreads] = 0;
        __syncthreads();
        x.count(hist, STEP, prefix, mask);
        __syncthreads();
        for (int n = t; n < evict_bins(STEP); n += kEvictThreads)
            if (hist[n]) atomicAdd(&own[2 + STEP * kEvictBins + n], hist[n]);
        return;
    }
    int above, equal;
    x.sums(prefix, above, equal);
    __syncthreads();
    if (lane == 0) {
        totals[wave][0] = above;
        totals[wave][1] = equal;
    }
    __syncthreads();
    int before = 0, same = 0, all = 0, equals = 0;
#pragma unroll
    for (int v = 0; v < kEvictWaves; ++v) {
        before += v < wave ? totals[v][0] : 0;
        same += v < wave ? totals[v][1] : 0;
        all += totals[v][0];
        equals += totals[v][1];
    }
    if constexpr (STEP == 3) {
        if (t == 0) {
            counts[2 * chunk] = all;
            counts[2 * chunk + 1] = equals;
        }
        return;
    }
    all = equals = 0;
    for (int c = lane; c < chunks; c += 64) {  // (at most 128)
        const int n = counts[2 * c], e = counts[2 * c + 1];
        all += n;
        equals += e;
        above = c < chunk ? n + (c < 64 ? 0 : above) : c < 64 ? 0 : above;
        equal = c < chunk ? e + (c < 64 ? 0 : equal) : c < 64 ? 0 : equal;
    }
    if (lane >= chunks) above = equal = 0;
    before += wave_sum(above);
    same += wave_sum(equal);
    all = wave_sum(all);
    equals = wave_sum(equals);
    x.write(a, bk, prefix, want, before + min(same, want), same, lane, 0, INT_MAX, nullptr);
    evict_rest(a, bk, all + min(equals, want), chunk * kEvictThreads + t, chunks * kEvictThreads);
}

// The kept slots' rows, by 256 threads.
__global__ void __launch_bounds__(256) paged_move_kernel(PagedEvict a, int row_bytes, int esize) {
    const int lanes = row_bytes / 16, rows = 256 / lanes, t = threadIdx.x;
    const int chunks = (a.keep + rows - 1) / rows, chunk = blockIdx.x % chunks, bk = blockIdx.x / chunks, b = bk / a.c.Hkv;
    const int n = chunk * rows + t / lanes, s = n < a.keep ? a.kept[(size_t)bk * a.keep + n] : -1;
    if (s >= 0) evict_move(a, b, bk - b * a.c.Hkv, s, n, t % lanes * 16, row_bytes, esize);
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

// The workgroups of the attention, and whether a unit may have several pieces.
// Larger batches: a piece a unit, as every workgroup reads all lengths to find its own.  One sequence of 30000 slots behind others of
// 400, us: 1024 sequences 67 (4 heads over 1 of 128), 303 (20 over 5), 1025 400, 485.
constexpr int kPagedMapped = 1024;
struct PagedShape {
    long long units, groups;
    int tiles;
    bool split, last;  // last: joined by a unit's last workgroup
};
PagedShape paged_shape(int B, int H, int Hkv, int cap, int type) {
    PagedShape p;
    const int G = H / Hkv, least = kWaves * (type == kPagedF32 ? 16 : 32);  // a piece's slots at least
    p.tiles = (G + 15) / 16;
    p.units = (long long)B * Hkv * p.tiles;
    const long long most = (cap + least - 1) / least;
    p.split = most > 1 && B <= kPagedMapped;
    // As many as run at once, two a CU, or twice that for two pieces a unit; past 512 units, pieces for sequences that have
    // more than a 512th of the work, no others.  Two pieces a unit / these / none, us: 128 sequences of 10 to 1500 slots (32 heads
    // over 8) 83 / 80 / 77, 1000 of 700 (4 over 1; each workgroup looks at every length) 98 / 69 / 59; one of 30000 among 255 of 400
    // (32 over 8) 127 with these, 428 with none, one among 63 (64 over 16) 87 / 416.
    p.groups = !p.split ? p.units : std::min(p.units * most, p.units <= 512 ? 512 * ((p.units + 255) / 256) : p.units + 512);
    // The last workgroup joins where no unit has more than 32 pieces, or 64 heads of pieces: a launch less on the host (3.5 us),
    // and on the GPU, us in two launches / one: 20 heads over 5, 1000 slots 6.4 + 3.2 / 8.6, 2000 6.3 + 3.8 / 9.0, 4000 (32 pieces of
    // 4 heads) 6.9 + 4.4 / 12.5; 32 over 2, 500 6.8 + 3.4 / 10.6; 16 over 1, 1000 (8 of 16) 6.8 + 3.8 / 11.3; 5 over 5, 8000 (63 of 1)
    // 9.8 + 4.2 / 15.7; one workgroup then reads what many would.
    const long long pieces = std::min(most, p.groups / ((long long)Hkv * p.tiles));
    p.last = p.split && B <= 64 && pieces <= 32 && pieces * std::min(G, 16) <= kLastMost;
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

// The workspace: sums [place][16][hd], (reference, sum of weights) [place][16][2], (place of the second piece, pieces) [unit], scores
// [B][KV head and tile of heads][tile of slots][head][slot] (a tile's in one piece: with a head's in one, writing them took
// 20 sequences of 3025 slots, 32 heads over 8, 47.5 us, so 46.7).
namespace {
// Where the launches' numbers start: some 44 bits that memory does not hold by itself.
unsigned long long paged_seed() {
    timespec t{};
    clock_gettime(CLOCK_REALTIME, &t);
    unsigned long long z = (unsigned long long)t.tv_sec * 1000000000ull + (unsigned long long)t.tv_nsec + ((unsigned long long)getpid() << 40);
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;  // (SplitMix64's finaliser)
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
}  // namespace
size_t paged_attention_workspace(int B, int H, int Hkv, int cap, int type, int hd, bool weights) {
    const PagedShape p = paged_shape(B, H, Hkv, cap, type);
    const size_t parts = (size_t)p.groups * 16;
    // (place of the second piece, pieces) or, instead, the ticket of a unit
    return 4 * ((p.split ? parts * hd : 0) + (p.split || weights ? parts * 2 + ((size_t)p.units * 2 + 3) / 4 * 4 : 0) +
                (weights ? (size_t)B * H * paged_even(cap) : 0));
}

// The weights are added by the workgroup that has a KV head's totals, a launch less, for up to 4096 scores a KV head and 2^17 in
// all (of the table's slots: the host does not know the lengths); a second launch otherwise.  us of a call in a row, and in a replayed
// graph, by the one | the other: 20 heads over 5 of 128 in bf16, 1 sequence of 1000 slots 11.7, 11.5 | 14.3, 10.0, 6 of up to 1000
// 12.0, 11.6 | 13.7, 10.5, 32 of 120 11.6, 8.7 | 14.0, 10.2; 12 heads over 12 of 64, 8 of up to 1000 12.1, 12.0 | 13.7, 11.1, 4 of up
// to 2000 14.2, 14.3 | 13.9, 11.1; past the limits 12 of up to 1000 15.2, 15.1 | 14.1, 13.4, 8 of up to 2000 (12 over 12) 16.0, 16.1 |
// 13.8, 13.5, 32 of up to 1000 18.8, 19.0 | 17.7, 17.6, 4 of 2000 18.8, 19.0 | 14.1, 13.9.  (Eager calls, whose launch costs the
// host more, decide.)
constexpr int kWeighHead = 1 << 12, kWeighAll = 1 << 17;

hipError_t launch_paged_attention(PagedAttn a, bool step, int type, int hd, void* work, hipStream_t s) {
    const int cap = a.c.P << a.c.shift;
    const PagedShape p = paged_shape(a.c.B, a.H, a.c.Hkv, cap, type);
    a.G = a.H / a.c.Hkv;
    a.tiles = p.tiles;
    a.scale = 1.44269504088896341f / sqrtf((float)hd);
    const size_t parts = (size_t)p.groups * 16;
    a.part = static_cast<float*>(work);
    a.ml = p.split || a.weights ? a.part + (p.split ? parts * hd : 0) : nullptr;
    a.units = reinterpret_cast<int2*>(a.ml + parts * 2);
    a.scores = a.weights ? a.ml + parts * 2 + ((size_t)p.units * 2 + 3) / 4 * 4 : nullptr;
    const bool few = p.tiles == 1 && (long long)cap * a.G <= kWeighHead && (long long)cap * a.G * p.units <= kWeighAll;
    a.whole = (p.last || !p.split) && (!a.weights || few);
    if (a.whole && p.split) {
        static std::atomic<unsigned long long> number{paged_seed()};
        const unsigned long long most = ~0ull >> kTicketBits;
        do a.nonce = number.fetch_add(1, std::memory_order_relaxed) & most;
        while (a.nonce == 0);
        a.tickets = reinterpret_cast<unsigned long long*>(a.units);
    }
    const long long groups = p.groups, joins = p.split && !a.whole ? (long long)a.c.B * a.H : 0;
    if (groups > kPagedMaxGroups) return hipErrorInvalidValue;
    a.groups = (int)groups;
    const bool wide = p.groups > 16 * p.units;  // a head's pieces by 16 waves
    const int nt = wide ? 1024 : 256, chunks = a.weights && !a.whole ? (cap + 4 * nt - 1) / (4 * nt) : 0;
    const long long second = joins + (long long)a.c.B * a.c.Hkv * chunks;
    if (second > kPagedMaxGroups) return hipErrorInvalidValue;
    paged_by_type(type, hd, [&](auto T, auto HD) {
        constexpr int t = decltype(T)::value, d = decltype(HD)::value;
        auto attend = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(64 * kWaves), 0, s, a); };
        // Keys and values that one workgroup reads, once, go past the caches.  us through them / past them (20 heads over 5 of 128,
        // bf16, three caches in turn): 131072 slots 67.5 / 59.5, 32 sequences of 100 to 4095 37.8 / 34.7; 32 of 16000, 16 heads over 1
        // 54.0 / 48.3.  Where tiles of heads share them, through the caches: 32 over 1 61.1 / 73.0, 64 95.6 / 126.  Pages that sequences
        // share are read past the caches too, as the host does not know the tables: 32 sequences over the same 4000 slots 32.7 / 49.6
        // (of their own 64.1 / 56.7), 500 11.5 / 12.4 (14.3 / 15.0).
        const bool once = p.tiles == 1;
        if (step) once ? attend(paged_attn_kernel<t, d, true, true>) : attend(paged_attn_kernel<t, d, true, false>);
        else once ? attend(paged_attn_kernel<t, d, false, true>) : attend(paged_attn_kernel<t, d, false, false>);
        if (!second) return;
        auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)second), dim3(nt), 0, s, a, type == kPagedF32 ? 16 : 32, (int)joins, chunks); };
        if (step) wide ? join(paged_join_kernel<d, true, 1024>) : join(paged_join_kernel<d, true, 256>);
        else wide ? join(paged_join_kernel<d, false, 1024>) : join(paged_join_kernel<d, false, 256>);
    });
    return hipGetLastError();
}

// What an eviction from caches of more than kEvictAlone slots needs beside its outputs.
size_t paged_evict_workspace(int B, int Hkv, int cap) {
    const size_t chunks = (cap + kEvictChunk - 1) / kEvictChunk;
    return cap <= kEvictAlone ? 0 : 4 * (size_t)B * Hkv * (kEvictWords + 2 * chunks);
}

hipError_t launch_paged_evict(const PagedEvict& a, int type, int hd, void* work, hipStream_t s) {
    const int esize = type == kPagedF32 ? 4 : 2, row = hd * esize, rows = 256 / (row / 16), cap = a.c.P << a.c.shift;
    const int chunks = (cap + kEvictChunk - 1) / kEvictChunk;
    const long long heads = (long long)a.c.B * a.c.Hkv, moves = heads * ((a.keep + rows - 1) / rows);
    if (moves > kPagedMaxGroups || heads * chunks > kPagedMaxGroups) return hipErrorInvalidValue;
    const dim3 block(kEvictThreads);
    if (cap <= kEvictAlone) {
        // as many workgroups a head as there are CUs for, but 64 rows each at least
        const int keep = std::min(a.keep, cap);
        const int parts = std::max((keep + kEvictShare - 1) / kEvictShare, (int)std::min<long long>((keep + 63) / 64, 256 / heads));
        const int share = (keep + parts - 1) / parts;
        if (heads * parts > kPagedMaxGroups) return hipErrorInvalidValue;
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)(heads * parts)), block, 0, s, a, parts, share, row, esize); };
        if (cap <= 4 * kEvictThreads) go(paged_select_kernel<4>);
        else if (cap <= 8 * kEvictThreads) go(paged_select_kernel<8>);
        else if (cap <= 16 * kEvictThreads) go(paged_select_kernel<16>);
        else go(paged_select_kernel<32>);
        return hipGetLastError();
    }
    int* const w = static_cast<int*>(work);
    const int words = kEvictWords + 2 * chunks;
    hipLaunchKernelGGL(paged_clear_kernel, dim3((unsigned)heads), block, 0, s, w, words);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)(heads * chunks)), block, 0, s, a, w, words, chunks); };
    go(paged_share_kernel<0>);
    go(paged_share_kernel<1>);
    go(paged_share_kernel<2>);
    go(paged_share_kernel<3>);
    go(paged_share_kernel<4>);
    hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)moves), dim3(256), 0, s, a, row, esize);
    return hipGetLastError();
}

}  // namespace rt
