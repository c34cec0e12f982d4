// Attention over a paged key-value cache: what the split form (attention.cu) and the prompt form (attention_tc.cu) share.
//
// Query token t of sequence b stands at position p = pos[b] + t and sees the keys j <= p of its sequence, with a window W only
// those with j > p - W or j < sinks:
//   o = sum_j e^(scale q.k_j - m) v_j / l,   m = max_j scale q.k_j,   l = sum_j e^(scale q.k_j - m),   lse = m + ln l
// Key j lives in row j % page_size of page table[b][j / page_size]. A token that sees nothing gets o = 0, lse = -inf; one whose
// keys lie on a page outside the pool, or whose position is beyond the table, gets NaN (nothing outside the pool is read).
#pragma once
#include <cmath>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "exl3_gemv_kernel.cuh"
#include "exl3_gemv_host.h"
#include "host_common.h"
#include "spans.h"
#include "../../include/ampstein_b200.h"

namespace amp {

constexpr int AT_MAX_POS = 1 << 30;            // positions are clamped to +- this (the table holds fewer)

struct AtSeq
{
    int first, count, row0;                    // position of the first query token, tokens, first row of q
};

// Tokens of sequence b with cu
__device__ __forceinline__ int at_count(const amp_attention_args& P, int b)
{
    const int row0 = max(0, min(P.cu[b], P.tokens));
    return max(row0, min(P.cu[b + 1], P.tokens)) - row0;
}

// Sequence b; each: tokens of every sequence without cu. Whatever pos and cu hold, the rows stay inside the tensors.
__device__ __forceinline__ AtSeq at_seq(const amp_attention_args& P, int b, int each)
{
    AtSeq s;
    const long long p = P.pos64 ? reinterpret_cast<const long long*>(P.pos)[b] : (long long) reinterpret_cast<const int*>(P.pos)[b];
    s.first = (int) max(-(long long) AT_MAX_POS, min((long long) AT_MAX_POS, p));
    if (P.cu)
    {
        s.row0 = max(0, min(P.cu[b], P.tokens));
        s.count = at_count(P, b);
    }
    else
    {
        s.count = each;
        s.row0 = b * each;
    }
    return s;
}

// Keys that some token of positions [first, first + count) sees: [0, a) and [lo, end), a <= lo <= end
struct AtKeys
{
    int a, lo, end;
    __device__ __forceinline__ int count() const { return a + end - lo; }
    __device__ __forceinline__ int key(int i) const { return i < a ? i : i - a + lo; }     // the i-th of them
};

__device__ __forceinline__ AtKeys at_keys(const amp_attention_args& P, int first, int count)
{
    AtKeys k;
    k.end = count > 0 ? max(0, min(first + count, P.max_pages * P.page_size)) : 0;
    k.lo = P.window ? min(k.end, max(0, first - P.window + 1)) : 0;
    k.a = P.window ? min(P.sinks, k.lo) : 0;
    return k;
}

// Division by what the host knows, exact for 0 <= j < 2^30: with 2^(s - 1) < d <= 2^s and mul = ceil(2^(30 + s) / d), j * mul / 2^(30 + s) is
// too large by less than j / 2^30 / d
struct AtDiv
{
    uint32_t mul, shift;
    __device__ __forceinline__ int of(int j) const { return (int) ((unsigned long long) (uint32_t) j * mul >> shift); }
};

inline AtDiv at_div(long d)
{
    int s = 0;
    while (s < 30 && (1l << s) < d) ++s;
    return { (uint32_t) (((1ull << (30 + s)) + d - 1) / d), (uint32_t) (30 + s) };
}

// Strides of the caches in pieces of 16 bytes (offsets inside a cache of up to 64 GB are 32-bit counts of them)
struct AtPages
{
    uint32_t k_page, k_row, v_page, v_row;
    AtDiv page_size;
    __device__ __forceinline__ int page_of(int j) const { return page_size.of(j); }
};

inline bool at_pages(const amp_attention_args& P, AtPages& g)
{
    auto fits = [&](long page, long row, long head) {
        const double most = 34359738368.0;     // values of 64 GB
        return page >= 0 && row >= 0 && head >= 0 && (double) (P.pages - 1) * page + (double) (P.page_size - 1) * row < most;
    };
    if (!fits(P.k_page, P.k_row, P.k_head) || !fits(P.v_page, P.v_row, P.v_head)) return false;
    g.k_page = (uint32_t) (P.k_page / 8); g.k_row = (uint32_t) (P.k_row / 8); g.v_page = (uint32_t) (P.v_page / 8); g.v_row = (uint32_t) (P.v_row / 8);
    g.page_size = at_div(P.page_size);
    return true;
}

// Of the keys counted through, the ones that the token at p sees: [0, n0) and [c1, c1 + len] (c1 out of reach: none)
__device__ __forceinline__ void at_row_keys(const amp_attention_args& P, const AtKeys& k, int p, int& n0, int& c1, int& len)
{
    n0 = P.window ? min(p + 1, P.sinks) : 0;
    c1 = P.window ? max(p - P.window + 1, k.lo) - k.lo + k.a : 0;
    len = p - k.lo + k.a - c1;
    if (len < 0) { c1 = 1 << 30; len = 0; }
}

// ... and a run of them, [from, to), that every token from p0 to p1 sees
__device__ __forceinline__ void at_whole_keys(const amp_attention_args& P, const AtKeys& k, int p0, int p1, int& from, int& to)
{
    to = min(k.count(), p0 - k.lo + k.a + 1);
    from = P.window ? k.a + max(0, p1 - P.window + 1 - k.lo) : 0;
}

__device__ __forceinline__ float at_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// odd: bits 15 and 31 are set for a value without a finite magnitude (its exponent is all ones: one more carries out of it), the others are
// of no matter
template <typename T> struct AtType;
template <> struct AtType<__half>
{
    // the largest weight is 2^weight_top, as far up as half goes, so that fewer fall below its normal range (2^-14) or out of it (2^-25), where
    // the sum in fp32 still counts them. 131000 keys 17 nats below one key: their share of the columns in which that one has no value,
    // 5.4e-3, is off by 2.4e-3 (prompts) and 5.9e-4 (few tokens) with 1 as the largest weight, by 7e-6 and 8e-7 so
    static constexpr float weight_top = 15.0f;
    static __device__ __forceinline__ uint32_t odd(uint32_t x) { return (x & 0x7c007c00u) + 0x04000400u; }
    static __device__ __forceinline__ float2 unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    static __device__ __forceinline__ __half from(float a) { return __float2half_rn(a); }
};
template <> struct AtType<__nv_bfloat16>
{
    static constexpr float weight_top = 0.0f;                // (fp32's range)
    static __device__ __forceinline__ uint32_t odd(uint32_t x) { return (x & 0x7f807f80u) + 0x00800080u; }
    static __device__ __forceinline__ float2 unpack(uint32_t x) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    static __device__ __forceinline__ __nv_bfloat16 from(float a) { return __float2bfloat16_rn(a); }
};

// What the weights of a row with the maximum m count from. (Far from 0 the maximum itself: there m - 15 is rounded, to m - 16 between 2^24 and
// 2^28, and 2^16 is infinite in half.)
template <typename T>
__device__ __forceinline__ float at_base(float m)
{
    return AtType<T>::weight_top == 0.0f || fabsf(m) > 1048576.0f ? m : m - AtType<T>::weight_top;
}

// An infinite or NaN value times the weight 0 of a row that does not see its key would be NaN. Where keys are seen by some rows only,
// such values are therefore taken out of the product, and added to the rows that do see them.
constexpr uint32_t AT_ODD = 0x80008000u;

template <typename T>
__device__ __forceinline__ uint32_t at_odd(uint4 v) { return (AtType<T>::odd(v.x) | AtType<T>::odd(v.y) | AtType<T>::odd(v.z) | AtType<T>::odd(v.w)) & AT_ODD; }

template <typename T>
__device__ __forceinline__ uint32_t at_even(uint32_t x) { return x & ~((AtType<T>::odd(x) >> 15 & 0x00010001u) * 0xffffu); }      // they are 0

__device__ __forceinline__ uint4 at_lds16(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

template <typename T>
__device__ __forceinline__ void at_sts16_even(uint32_t addr, uint4 v)
{
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                 :: "r"(addr), "r"(at_even<T>(v.x)), "r"(at_even<T>(v.y)), "r"(at_even<T>(v.z)), "r"(at_even<T>(v.w)) : "memory");
}

// 16 bytes to shared memory, or zeros
__device__ __forceinline__ void at_copy16(uint32_t dst, const void* src, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

// What a finished row's sums are multiplied by, 1 / l (a position beyond the table has keys that cannot be found: NaN)
__device__ __forceinline__ float at_factor(const amp_attention_args& P, int p, float l)
{
    return p >= P.max_pages * P.page_size ? NAN : (l == 0.0f ? 0.0f : 1.0f / l);
}

// Stores four or eight values of a finished row (f: at_factor), and with the first of them its lse. m counts in powers of two.
template <typename T>
__device__ __forceinline__ T* at_out(const amp_attention_args& P, const AtSeq& s, int tok, int head, int c, float f, float m, float l)
{
    if (c == 0 && P.lse)
        P.lse[(long long) (s.row0 + tok) * P.heads + head] = f != f ? NAN : (l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f);
    return reinterpret_cast<T*>(P.out) + (long long) (s.row0 + tok) * P.out_token + (long long) head * P.out_head + c;
}

template <typename T>
__device__ __forceinline__ void at_store(const amp_attention_args& P, const AtSeq& s, int tok, int head, int c, float4 x, float m, float l)
{
    const float f = at_factor(P, s.first + tok, l);
    *reinterpret_cast<uint2*>(at_out<T>(P, s, tok, head, c, f, m, l)) = make_uint2(AtType<T>::pack(x.x * f, x.y * f), AtType<T>::pack(x.z * f, x.w * f));
}

template <typename T>
__device__ __forceinline__ void at_store8(const amp_attention_args& P, const AtSeq& s, int tok, int head, int c, float4 x, float4 y, float f, float m, float l)
{
    *reinterpret_cast<uint4*>(at_out<T>(P, s, tok, head, c, f, m, l)) =
        make_uint4(AtType<T>::pack(x.x * f, x.y * f), AtType<T>::pack(x.z * f, x.w * f), AtType<T>::pack(y.x * f, y.y * f), AtType<T>::pack(y.z * f, y.w * f));
}

}  // namespace amp
