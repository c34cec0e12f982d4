// Rotary positions of queries and keys, and the write of new keys and values into a paged cache, in one launch: what stands
// between the q|k|v projections and the attention.
//
// Bound by memory where there are many tokens (every head is read and written once), by the launch where there is one. A CTA
// takes one token: it requests its heads first, makes the token's rot / 2 pairs of cos and sin under those loads (once, for all
// heads), then turns and stores. A thread keeps one place inside the head, 16 values wide, through all its heads: its eight
// cos and sin stay in registers.
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

// Where head h of the token (queries, then keys, then values) is read and written; to == null: it is not stored
template <typename T>
struct RopeHead
{
    const T* from;
    T* to;
};

template <typename T>
__device__ __forceinline__ RopeHead<T> rope_head(const amp_rope_args& P, int n, int h, long long kc, long long vc)
{
    RopeHead<T> r;
    if (h < P.heads)
    {
        r.from = reinterpret_cast<const T*>(P.q) + (long long) n * P.q_token + (long long) h * P.q_head;
        r.to = reinterpret_cast<T*>(P.q_out) + (long long) n * P.out_token + (long long) h * P.out_head;
        return r;
    }
    h -= P.heads;
    if (h < P.kv_heads)
    {
        r.from = reinterpret_cast<const T*>(P.k) + (long long) n * P.k_token + (long long) h * P.k_head;
        r.to = kc < 0 ? nullptr : reinterpret_cast<T*>(P.k_cache) + kc + (long long) h * P.kc_head;
        return r;
    }
    h -= P.kv_heads;
    r.from = reinterpret_cast<const T*>(P.v) + (long long) n * P.v_token + (long long) h * P.v_head;
    r.to = vc < 0 ? nullptr : reinterpret_cast<T*>(P.v_cache) + vc + (long long) h * P.vc_head;
    return r;
}

// VEC: 16 bytes at a time; else value by value (a rotated part or a head that is not a multiple of 16 values, or other alignments)
template <typename T, bool VEC>
__global__ __launch_bounds__(ROPE_THREADS)
void rope_kernel(const amp_rope_args P, int pdl)
{
    __shared__ __align__(16) float2 s_cs[ROPE_MAX_DIM / 2];
    __shared__ int s_seq;
    const int t = threadIdx.x, n = blockIdx.x;
    if (pdl) { pdl_wait(); pdl_launch_dependents(); }

    int b, first_row;
    if (P.cu)
    {
        if (t == 0) s_seq = -1;
        __syncthreads();
        for (int i = t; i < P.seqs; i += ROPE_THREADS) if (P.cu[i] <= n && n < P.cu[i + 1]) s_seq = i;
        __syncthreads();
        b = s_seq;
        if (b < 0) return;                                   // behind the last sequence
        first_row = P.cu[b];
    }
    else
    {
        const int each = P.tokens / P.seqs;
        b = n / each;
        first_row = b * each;
    }
    const long long p = (P.pos64 ? reinterpret_cast<const long long*>(P.pos)[b] : (long long) reinterpret_cast<const int*>(P.pos)[b]) + (n - first_row);

    long long kc = -1, vc = -1;
    if (P.k && p >= 0 && p < (long long) P.max_pages * P.page_size)
    {
        const int pg = (int) p / P.page_size, row = (int) p - pg * P.page_size, page = P.table[(long long) b * P.table_row + pg];
        if (page >= 0 && page < P.pages)
        {
            kc = page * P.kc_page + row * P.kc_row;
            vc = page * P.vc_page + row * P.vc_row;
        }
    }
    const int total = P.heads + (P.k ? 2 * P.kv_heads : 0), rotated = P.heads + (P.k ? P.kv_heads : 0);

    if constexpr (VEC)
    {
        const int places = P.dim / 16, step = ROPE_THREADS / places, turning = P.rot / 16;
        const int c = t % places, h0 = t / places;
        const bool turns = c < turning;
        const int at0 = 8 * (turns && !P.interleaved ? c : 2 * c), at1 = 8 * (turns && !P.interleaved ? c + turning : 2 * c + 1);
        const bool mine = h0 < step;                         // (128 is not a multiple of every width)
        constexpr int BATCH = 4;
        float2 cs[8];
        bool have = false;
        for (int h = h0; ; h += BATCH * step)
        {
            uint4 x[BATCH], y[BATCH];
            #pragma unroll
            for (int i = 0; i < BATCH; ++i)
            {
                if (!mine || h + i * step >= total) continue;
                const RopeHead<T> r = rope_head<T>(P, n, h + i * step, kc, vc);
                x[i] = *reinterpret_cast<const uint4*>(r.from + at0);
                y[i] = *reinterpret_cast<const uint4*>(r.from + at1);
            }
            if (!have)
            {
                for (int i = t; i < P.rot / 2; i += ROPE_THREADS) s_cs[i] = rope_turn((double) p, P.inv_freq[i], P.mscale);
                __syncthreads();
                if (turns)
                {
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) cs[i] = s_cs[8 * c + i];
                }
                have = true;
            }
            if (!mine || h >= total) break;
            #pragma unroll
            for (int i = 0; i < BATCH; ++i)
            {
                if (h + i * step >= total) continue;
                const RopeHead<T> r = rope_head<T>(P, n, h + i * step, kc, vc);
                if (!r.to) continue;
                if (turns && h + i * step < rotated) rope_pairs<T>(x[i], y[i], cs, P.interleaved);
                *reinterpret_cast<uint4*>(r.to + at0) = x[i];
                *reinterpret_cast<uint4*>(r.to + at1) = y[i];
            }
        }
    }
    else
    {
        for (int i = t; i < P.rot / 2; i += ROPE_THREADS) s_cs[i] = rope_turn((double) p, P.inv_freq[i], P.mscale);
        __syncthreads();
        const int half = P.rot / 2, each = half + P.dim - P.rot;        // a thread owns both values of a pair: q_out may be q
        for (int i = t; i < total * each; i += ROPE_THREADS)
        {
            const int h = i / each, e = i - h * each;
            const RopeHead<T> r = rope_head<T>(P, n, h, kc, vc);
            if (!r.to) continue;
            if (e >= half) { r.to[P.rot + e - half] = r.from[P.rot + e - half]; continue; }
            const int a = P.interleaved ? 2 * e : e, z = P.interleaved ? 2 * e + 1 : e + half;
            const T u = r.from[a], v = r.from[z];
            if (h >= rotated) { r.to[a] = u; r.to[z] = v; continue; }
            const float uf = rope_value(u), vf = rope_value(v);
            const float2 cs = s_cs[e];
            r.to[a] = AtType<T>::from(uf * cs.x - vf * cs.y);
            r.to[z] = AtType<T>::from(vf * cs.x + uf * cs.y);
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
    return cuda_rc(vec ? cudaLaunchKernelEx(&cfg, rope_kernel<T, true>, (const amp_rope_args) P, g_pdl)
                       : cudaLaunchKernelEx(&cfg, rope_kernel<T, false>, (const amp_rope_args) P, g_pdl), "rope launch");
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
    uintptr_t ptrs = (uintptr_t) P.q | (uintptr_t) P.q_out;
    long strides = P.q_token | P.q_head | P.out_token | P.out_head;
    if (P.k || P.v || P.k_cache || P.v_cache || P.table)
    {
        AMP_REQUIRE(P.k && P.v && P.k_cache && P.v_cache && (P.table || P.max_pages == 0), "rope: k, v, both caches and the table go together");
        AMP_REQUIRE(P.kv_heads > 0 && P.kv_heads <= 1024 && P.pages > 0 && P.page_size > 0 && P.max_pages >= 0 && (long long) P.max_pages * P.page_size <= AT_MAX_POS,
                    "rope: page sizes (up to 2^30 positions per sequence)");
        ptrs |= (uintptr_t) P.k | (uintptr_t) P.v | (uintptr_t) P.k_cache | (uintptr_t) P.v_cache;
        strides |= P.k_token | P.k_head | P.v_token | P.v_head | P.kc_page | P.kc_row | P.kc_head | P.vc_page | P.vc_row | P.vc_head;
    }
    AMP_REQUIRE((ptrs & 1) == 0, "rope: misaligned pointer");
    const bool vec = P.rot % 16 == 0 && P.dim % 16 == 0 && P.dim <= 16 * ROPE_THREADS && (ptrs & 15) == 0 && (strides & 7) == 0;
    return P.bf16 ? rope_launch<__nv_bfloat16>(P, vec, stream) : rope_launch<__half>(P, vec, stream);
}
