// Rotary positions of queries and keys, and the write of new keys and values into a paged cache, in one launch: what stands
// between the q|k|v projections and the attention.
//
// Bound by memory where there are many tokens (every head is read and written once), by the launch where there is one. A CTA
// takes one token: it requests its heads first, makes the token's rot / 2 pairs of cos and sin under those loads (once, for all
// heads), then turns and stores. A thread keeps one place inside the head, 16 values wide, through all its heads: its eight
// cos and sin stay in registers.
//
// Measured: 2.4 us for one token of 32 + 2 x 8 heads of 128 values; 2047 tokens of five sequences, 48 + 2 x 8 heads, 15.3 us (4.4 TB/s
// in and out, 0.68 of the measured copy rate: a CTA's chain of positions, table entry, cos and sin, store is not hidden whole).
//
// The angle p * inv_freq is taken modulo a turn in fp64: at p = 10^6 an fp32 product is off by 0.06 rad.
#include "attention.cuh"

namespace amp {

constexpr int ROPE_THREADS = 128;
constexpr int ROPE_MAX_DIM = 1024;

__device__ __forceinline__ float2 rope_turn(double p, float freq, float mscale)
{
    const double turns = p * (double) freq * 0.15915494309189535;
    float s, c;
    sincospif((float) (2.0 * (turns - rint(turns))), &s, &c);
    return make_float2(c * mscale, s * mscale);
}

template <typename T> __device__ __forceinline__ float2 rope_unpack(uint32_t x);
template <> __device__ __forceinline__ float2 rope_unpack<__half>(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
template <> __device__ __forceinline__ float2 rope_unpack<__nv_bfloat16>(uint32_t x) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x)); }

__device__ __forceinline__ float rope_value(__half x) { return __half2float(x); }
__device__ __forceinline__ float rope_value(__nv_bfloat16 x) { return __bfloat162float(x); }

// Eight pairs: (a, b) hold the first and the second values of them (half layout), or the pairs one after the other (interleaved)
template <typename T>
__device__ __forceinline__ void rope_pairs(uint4& a, uint4& b, const float2 (&cs)[8], bool interleaved)
{
    uint32_t* const x = reinterpret_cast<uint32_t*>(&a);
    uint32_t* const y = reinterpret_cast<uint32_t*>(&b);
    if (interleaved)
    {
        #pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const float2 u = rope_unpack<T>(x[i]), v = rope_unpack<T>(y[i]);
            x[i] = AtType<T>::pack(u.x * cs[i].x - u.y * cs[i].y, u.y * cs[i].x + u.x * cs[i].y);
            y[i] = AtType<T>::pack(v.x * cs[i + 4].x - v.y * cs[i + 4].y, v.y * cs[i + 4].x + v.x * cs[i + 4].y);
        }
    }
    else
    {
        #pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const float2 u = rope_unpack<T>(x[i]), v = rope_unpack<T>(y[i]), c0 = cs[2 * i], c1 = cs[2 * i + 1];
            x[i] = AtType<T>::pack(u.x * c0.x - v.x * c0.y, u.y * c1.x - v.y * c1.y);
            y[i] = AtType<T>::pack(v.x * c0.x + u.x * c0.y, v.y * c1.x + u.y * c1.y);
        }
    }
}

// Where head h of token n (queries, then keys, then values) is read, and written; null: it is not stored
template <typename T>
__device__ __forceinline__ const T* rope_from(const amp_rope_args& P, int n, int h)
{
    if (h < P.heads) return reinterpret_cast<const T*>(P.q) + (long long) n * P.q_token + (long long) h * P.q_head;
    h -= P.heads;
    if (h < P.kv_heads) return reinterpret_cast<const T*>(P.k) + (long long) n * P.k_token + (long long) h * P.k_head;
    return reinterpret_cast<const T*>(P.v) + (long long) n * P.v_token + (long long) (h - P.kv_heads) * P.v_head;
}

template <typename T>
__device__ __forceinline__ T* rope_to(const amp_rope_args& P, int n, int h, long long kc, long long vc)
{
    if (h < P.heads) return reinterpret_cast<T*>(P.q_out) + (long long) n * P.out_token + (long long) h * P.out_head;
    h -= P.heads;
    if (kc < 0) return nullptr;
    if (h < P.kv_heads) return reinterpret_cast<T*>(P.k_cache) + kc + (long long) h * P.kc_head;
    return reinterpret_cast<T*>(P.v_cache) + vc + (long long) (h - P.kv_heads) * P.vc_head;
}

// The arguments, and what a CTA divides by (products: one token 2.55 -> 2.43 us, 2048 level)
struct RopePlan
{
    amp_rope_args P;
    AtDiv by_page, by_each, by_places;
    int each, pdl;
};

// VEC: 16 bytes at a time; else value by value (a rotated part or a head that is not a multiple of 16 values, or other alignments)
template <typename T, bool VEC>
__global__ __launch_bounds__(ROPE_THREADS)
void rope_kernel(const RopePlan S)
{
    const amp_rope_args& P = S.P;
    __shared__ __align__(16) float2 s_cs[ROPE_MAX_DIM / 2];
    __shared__ int s_seq;
    const int t = threadIdx.x, n = blockIdx.x;
    if (S.pdl) { pdl_wait(); pdl_launch_dependents(); }
    const int total = P.heads + (P.k ? 2 * P.kv_heads : 0), rotated = P.heads + (P.k ? P.kv_heads : 0);

    // a thread's place in every head, and its first heads: requested before anything else is known of the token
    constexpr int BATCH = 4;                                 // (and of the value-by-value form)
    const int places = P.dim / 16, step = VEC ? S.by_places.of(ROPE_THREADS) : 0, turning = P.rot / 16;
    const int h0 = VEC ? S.by_places.of(t) : 0, c = VEC ? t - h0 * places : 0;
    const bool turns = c < turning, mine = h0 < step;        // (128 is not a multiple of every width)
    const int at0 = 8 * (turns && !P.interleaved ? c : 2 * c), at1 = 8 * (turns && !P.interleaved ? c + turning : 2 * c + 1);
    uint4 x[BATCH], y[BATCH];
    auto fetch = [&](int h) {
        #pragma unroll
        for (int i = 0; i < BATCH; ++i)
        {
            if (!mine || h + i * step >= total) continue;
            const T* from = rope_from<T>(P, n, h + i * step);
            x[i] = *reinterpret_cast<const uint4*>(from + at0);
            y[i] = *reinterpret_cast<const uint4*>(from + at1);
        }
    };
    if constexpr (VEC) fetch(h0);

    int b = n, first_row;
    long long p;
    auto position = [&](int i) { return P.pos64 ? reinterpret_cast<const long long*>(P.pos)[i] : (long long) reinterpret_cast<const int*>(P.pos)[i]; };
    if (P.cu && P.seqs <= 32)
    {
        // every warp by itself: a sequence per lane, its position on the way with its rows
        const int lane = t & 31;
        int lo = 0, hi = 0;
        p = 0;
        if (lane < P.seqs) { lo = P.cu[lane]; hi = P.cu[lane + 1]; p = position(lane); }
        const uint32_t hit = __ballot_sync(0xffffffffu, lo <= n && n < hi);
        if (!hit) return;                                    // behind the last sequence
        b = __ffs(hit) - 1;
        first_row = __shfl_sync(0xffffffffu, lo, b);
        p = __shfl_sync(0xffffffffu, p, b);
    }
    else if (P.cu)
    {
        if (t == 0) s_seq = -1;
        __syncthreads();
        for (int i = t; i < P.seqs; i += ROPE_THREADS) if (P.cu[i] <= n && n < P.cu[i + 1]) s_seq = i;
        __syncthreads();
        b = s_seq;
        if (b < 0) return;
        first_row = P.cu[b];
        p = position(b);
    }
    else
    {
        b = S.by_each.of(n);
        first_row = b * S.each;
        p = position(b);
    }
    p += n - first_row;
    int page = -1, row = 0;
    if (P.k && p >= 0 && p < (long long) P.max_pages * P.page_size)
    {
        const int pg = S.by_page.of((int) p);
        row = (int) p - pg * P.page_size;
        page = P.table[(long long) b * P.table_row + pg];
    }
    // (under the table's entry)
    for (int i = t; i < P.rot / 2; i += ROPE_THREADS) s_cs[i] = rope_turn((double) p, P.inv_freq[i], P.mscale);
    __syncthreads();
    const bool stored = page >= 0 && page < P.pages;
    const long long kc = stored ? page * P.kc_page + row * P.kc_row : -1, vc = stored ? page * P.vc_page + row * P.vc_row : -1;

    if constexpr (VEC)
    {
        if (!mine) return;
        float2 cs[8];
        if (turns)
        {
            #pragma unroll
            for (int i = 0; i < 8; ++i) cs[i] = s_cs[8 * c + i];
        }
        for (int h = h0; h < total; h += BATCH * step)
        {
            if (h > h0) fetch(h);
            #pragma unroll
            for (int i = 0; i < BATCH; ++i)
            {
                if (h + i * step >= total) continue;
                T* to = rope_to<T>(P, n, h + i * step, kc, vc);
                if (!to) continue;
                if (turns && h + i * step < rotated) rope_pairs<T>(x[i], y[i], cs, P.interleaved);
                *reinterpret_cast<uint4*>(to + at0) = x[i];
                *reinterpret_cast<uint4*>(to + at1) = y[i];
            }
        }
    }
    else
    {
        // a thread owns both values of a pair: q_out may be q. Four at a time, all read before the first is turned
        const int half = P.rot / 2, each = half + P.dim - P.rot;
        for (int i0 = t; i0 < total * each; i0 += BATCH * ROPE_THREADS)
        {
            T u[BATCH], v[BATCH];
            #pragma unroll
            for (int k = 0; k < BATCH; ++k)
            {
                const int i = i0 + k * ROPE_THREADS, h = i / each, e = i - h * each;
                if (i >= total * each) continue;
                const T* from = rope_from<T>(P, n, h);
                u[k] = from[e >= half ? P.rot + e - half : P.interleaved ? 2 * e : e];
                if (e < half) v[k] = from[P.interleaved ? 2 * e + 1 : e + half];
            }
            #pragma unroll
            for (int k = 0; k < BATCH; ++k)
            {
                const int i = i0 + k * ROPE_THREADS, h = i / each, e = i - h * each;
                T* to = i < total * each ? rope_to<T>(P, n, h, kc, vc) : nullptr;
                if (!to) continue;
                if (e >= half) { to[P.rot + e - half] = u[k]; continue; }
                if (h < rotated)
                {
                    const float uf = rope_value(u[k]), vf = rope_value(v[k]);
                    const float2 cs = s_cs[e];
                    u[k] = AtType<T>::from(uf * cs.x - vf * cs.y);
                    v[k] = AtType<T>::from(vf * cs.x + uf * cs.y);
                }
                to[P.interleaved ? 2 * e : e] = u[k];
                to[P.interleaved ? 2 * e + 1 : e + half] = v[k];
            }
        }
    }
}

template <typename T>
static int rope_launch(const amp_rope_args& P, bool vec, cudaStream_t stream)
{
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(P.tokens, 1, 1);
    cfg.blockDim = dim3(ROPE_THREADS, 1, 1);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = g_pdl ? 1 : 0;
    RopePlan S;
    S.P = P; S.each = max(1, P.tokens / P.seqs); S.pdl = g_pdl;
    S.by_page = at_div(max(1, P.page_size)); S.by_each = at_div(S.each); S.by_places = at_div(max(1, P.dim / 16));
    return cuda_rc(vec ? cudaLaunchKernelEx(&cfg, rope_kernel<T, true>, (const RopePlan) S)
                       : cudaLaunchKernelEx(&cfg, rope_kernel<T, false>, (const RopePlan) S), "rope launch");
}

}  // namespace amp

using namespace amp;

AMP_API int amp_b200_rope(const amp_rope_args* args, cudaStream_t stream)
{
    AMP_REQUIRE(args, "rope: null arguments");
    const amp_rope_args& P = *args;
    if (P.tokens == 0 || P.seqs == 0) return 0;
    AMP_REQUIRE(P.q && P.q_out && P.pos && (P.inv_freq || P.rot == 0), "rope: null pointer");
    AMP_REQUIRE(P.tokens > 0 && P.seqs > 0 && P.tokens <= (1 << 24) && P.seqs <= (1 << 20), "rope: %d tokens of %d sequences", P.tokens, P.seqs);
    AMP_REQUIRE(P.cu || P.tokens % P.seqs == 0, "rope: %d tokens do not divide into %d sequences", P.tokens, P.seqs);
    AMP_REQUIRE(P.dim > 0 && P.dim <= ROPE_MAX_DIM && P.rot >= 0 && P.rot <= P.dim && P.rot % 2 == 0 && P.heads > 0 && P.heads <= 1024,
                "rope: heads of %d values (up to %d), an even number of them rotated, not %d", P.dim, ROPE_MAX_DIM, P.rot);
    const Span q(P.q, P.dim * 2l, { { P.tokens, P.q_token * 2 }, { P.heads, P.q_head * 2 } }), out(P.q_out, P.dim * 2l, { { P.tokens, P.out_token * 2 }, { P.heads, P.out_head * 2 } });
    AMP_REQUIRE(q.same(out) || apart(q, out), "rope: q_out overlaps q (it may be q itself)");
    uintptr_t ptrs = (uintptr_t) P.q | (uintptr_t) P.q_out;
    long strides = P.q_token | P.q_head | P.out_token | P.out_head;
    if (P.k || P.v || P.k_cache || P.v_cache || P.table)
    {
        AMP_REQUIRE(P.k && P.v && P.k_cache && P.v_cache && (P.table || P.max_pages == 0), "rope: k, v, both caches and the table go together");
        AMP_REQUIRE(P.kv_heads > 0 && P.kv_heads <= 1024 && P.pages > 0 && P.page_size > 0 && P.max_pages >= 0 && (long long) P.max_pages * P.page_size <= AT_MAX_POS,
                    "rope: page sizes (up to 2^30 positions per sequence)");
        const Span k(P.k, P.dim * 2l, { { P.tokens, P.k_token * 2 }, { P.kv_heads, P.k_head * 2 } }), v(P.v, P.dim * 2l, { { P.tokens, P.v_token * 2 }, { P.kv_heads, P.v_head * 2 } });
        const Span kc(P.k_cache, P.dim * 2l, { { P.pages, P.kc_page * 2 }, { P.page_size, P.kc_row * 2 }, { P.kv_heads, P.kc_head * 2 } });
        const Span vc(P.v_cache, P.dim * 2l, { { P.pages, P.vc_page * 2 }, { P.page_size, P.vc_row * 2 }, { P.kv_heads, P.vc_head * 2 } });
        for (const Span* w : { &out, &kc, &vc })
            AMP_REQUIRE(apart(*w, k) && apart(*w, v), "rope: k or v overlaps %s", w == &out ? "q_out" : "a cache");
        AMP_REQUIRE(apart(kc, vc) && apart(kc, q) && apart(vc, q) && apart(kc, out) && apart(vc, out), "rope: a cache overlaps the other one, q or q_out");
        ptrs |= (uintptr_t) P.k | (uintptr_t) P.v | (uintptr_t) P.k_cache | (uintptr_t) P.v_cache;
        strides |= P.k_token | P.k_head | P.v_token | P.v_head | P.kc_page | P.kc_row | P.kc_head | P.vc_page | P.vc_row | P.vc_head;
    }
    AMP_REQUIRE((ptrs & 1) == 0, "rope: misaligned pointer");
    const bool vec = P.rot % 16 == 0 && P.dim % 16 == 0 && P.dim <= 16 * ROPE_THREADS && (ptrs & 15) == 0 && (strides & 7) == 0;
    return P.bf16 ? rope_launch<__nv_bfloat16>(P, vec, stream) : rope_launch<__half>(P, vec, stream);
}
