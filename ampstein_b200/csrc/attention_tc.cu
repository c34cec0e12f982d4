// Attention of prompt chunks over a paged key-value cache on the tensor cores (tcgen05, accumulators in tensor memory).
//
// The query heads that share a key-value head, times a sequence's new tokens, are the rows of one problem (row = token * group + head),
// so that a tile of 128 rows spans few tokens, keys are fetched once for the whole group, and a short chunk fills its tiles. A CTA takes
// NQ tiles of 128 rows (one at 256 values per head, and where a tile sees few keys; else two) and walks the keys that its tokens see in tiles of KB:
//   S = Q K^T     both operands K-major in shared memory, S (128 x KB fp32) in tensor memory
//   P = 2^(scale S - m), a row per thread: no exchange between threads; P goes back over S, in the operands' type
//   O += P V      P from tensor memory, V as it lies in the cache (N-major), O (128 x D fp32) in tensor memory
// With two tiles the tensor cores multiply for one while the other's softmax runs; with one tile S has two buffers, and the next
// Q K^T runs under the softmax. m moves only when a row's maximum has grown by more than 2^8 (with fp16 the weights begin 2^7 above 1, and stay
// below 2^15 and a rounding), so that O is rarely scaled again. Where the grid leaves SMs idle the keys of a tile are cut into
// slices, whose parts a second kernel joins in order.
//
// Warps: four per row tile do the softmax (a thread a row, the warp's quarter of tensor memory), then one issues the MMAs, three load
// keys and values by 16-byte asynchronous copies (a page of any size, strides of any kind).
//
// What bounds it (8192 tokens, 32 query heads on 8 key-value heads of 128 values, fp16): 495 us in bursts of four, 1110 TFLOP/s, 0.67 of the
// measured burst rate (577 among other calls, under the power cap: 950, 0.68 of the measured sustained rate); tensor and exponential pipe active in 54 % of the cycles each. A row tile's chain, scores read 0.15 us, maximum 0.2, weights
// 0.75, its P V and the next Q K^T 0.5, is longer than the other tile's MMAs, and the rows of a page reach shared memory through three
// warps at about 0.8 us per tile of keys or values. Measured and taken back: seven loading warps (registers of the softmax), TMA gathers of
// four rows (67 cycles each: 1121 us) and TMA boxes of a page's rows (level), two threads per row (544), a maximum that lags a
// half tile (499), 64 keys with two buffers of S for two row tiles (683). At 64 values the exponentials bind, and a quarter of them
// goes through the polynomial (397 -> 376 us for 8192 tokens; at 128 values 490 -> 504).
//
// Every mbarrier wait is bounded: a role whose wait ran out hands nothing over any more, whatever depends on it runs out too, nothing
// is stored (slices: their rows become NaN), the status word is set, and the CTA leaves when its copies and MMAs are done.
#include "attention_tc.cuh"
#include <mutex>

namespace amp {

__device__ int g_at_status;

constexpr unsigned AT_SPIN_LIMIT = 1u << 21;   // looks at a barrier before a wait is declared lost (a look lasts up to 4 us)
constexpr int TA_LOADERS = 3;                  // warps that load keys and values
constexpr int TA_AHEAD = 2;                    // tiles on their way when the next is requested
template <int D> constexpr int ta_poly = D == 64 ? 1 : 0;     // pairs of four whose exponentials are a polynomial's
constexpr float TA_FAR = 1048576.0f;           // a maximum beyond this (in powers of two) is off by more than 1/16 when it is rounded
constexpr float TA_SLACK = 8.0f;               // powers of two that a row's maximum may grow before O is scaled again

__device__ __forceinline__ bool ta_wait(uint32_t bar, uint32_t parity)
{
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\t"
        "mov.u32 n, %3;\n"
        "$TA_POLL_%=:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@p bra $TA_DONE_%=;\n\t"
        "sub.u32 n, n, 1;\n\t"
        "setp.ne.u32 q, n, 0;\n\t"
        "@q bra $TA_POLL_%=;\n"
        "$TA_DONE_%=:\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r) : "r"(bar), "r"(parity), "n"(AT_SPIN_LIMIT) : "memory");
    return r != 0;
}

__device__ __forceinline__ void ta_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}

__device__ __forceinline__ void ta_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}

__device__ __forceinline__ bool ta_elect()
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// Shared-memory descriptor of an operand in 128-byte swizzle: rows of 128 bytes, groups of eight rows 1024 bytes apart; block: bytes between
// the blocks of 64 values along N (N-major operands only)
__device__ __forceinline__ uint64_t ta_desc(uint32_t addr, uint32_t block)
{
    return (uint64_t) ((addr & 0x3ffff) >> 4) | ((uint64_t) (block >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// kind::f16 instruction descriptor: fp32 accumulator, 128 x n, A K-major, B K-major or N-major
__host__ __device__ constexpr uint32_t ta_idesc(int n, bool bf16, bool b_n_major)
{
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_n_major ? 1u : 0u) << 16) | ((uint32_t) (n >> 3) << 17) | (8u << 24);
}

__device__ __forceinline__ void ta_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ void ta_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

#define TA_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define TA_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 columns of the thread's row of tensor memory
__device__ __forceinline__ void ta_ld32(uint32_t addr, uint32_t* r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : TA_R8(r, 0), TA_R8(r, 8), TA_R8(r, 16), TA_R8(r, 24) : "r"(addr) : "memory");
}

__device__ __forceinline__ void ta_st32(uint32_t addr, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
                 "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 :: "r"(addr), TA_W8(r, 0), TA_W8(r, 8), TA_W8(r, 16), TA_W8(r, 24) : "memory");
}
__device__ __forceinline__ void ta_ld16(uint32_t addr, uint32_t* r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : TA_R8(r, 0), TA_R8(r, 8) : "r"(addr) : "memory");
}

__device__ __forceinline__ void ta_st16(uint32_t addr, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 :: "r"(addr), TA_W8(r, 0), TA_W8(r, 8) : "memory");
}
#undef TA_R8
#undef TA_W8

__device__ __forceinline__ void ta_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ta_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ta_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ta_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ta_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 2^y of two values without the exponential unit, which has 16 results a clock for the SM and would be busy as long as the tensor
// cores: y = i + f with i the nearest whole number, 2^f on [-1/2, 1/2] by a polynomial of degree 5 (minimax in the relative error, by
// Remez exchange: 7.5e-8, 1.5e-7 with its coefficients in fp32, 2.1e-7 as it is evaluated here), 2^i through the exponent field. Below 2^-126.5: 0 (the field is 0); a NaN stays one. y <= 127.
__device__ __forceinline__ float2 ta_exp2_pair(f32x2 y2)
{
    float2 y = unpack_f32x2(y2);
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(y.x));      // -127
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(y.y));
    y2 = pack_f32x2(y.x, y.y);
    constexpr float MAGIC = 12582912.0f + 127.0f;            // 1.5 2^23: the sum's last bits are i + 127
    const f32x2 t = add_f32x2(y2, pack_f32x2(MAGIC, MAGIC));
    const f32x2 f = fma_f32x2(add_f32x2(t, pack_f32x2(-MAGIC, -MAGIC)), pack_f32x2(-1.0f, -1.0f), y2);
    f32x2 p = pack_f32x2(0x1.5c08e6p-10f, 0x1.5c08e6p-10f);
    p = fma_f32x2(p, f, pack_f32x2(0x1.3d0c52p-7f, 0x1.3d0c52p-7f));
    p = fma_f32x2(p, f, pack_f32x2(0x1.c6b6e4p-5f, 0x1.c6b6e4p-5f));
    p = fma_f32x2(p, f, pack_f32x2(0x1.ebf918p-3f, 0x1.ebf918p-3f));
    p = fma_f32x2(p, f, pack_f32x2(0x1.62e428p-1f, 0x1.62e428p-1f));
    p = fma_f32x2(p, f, pack_f32x2(0x1.000002p+0f, 0x1.000002p+0f));
    const float2 u = unpack_f32x2(t);
    return unpack_f32x2(mul_f32x2(p, pack_f32x2(__uint_as_float(__float_as_uint(u.x) << 23), __uint_as_float(__float_as_uint(u.y) << 23))));
}

// Sequence of the x-th row tile of the call, and the tile in it; false: there is none. By one warp.
struct TaPlace
{
    AtSeq s;
    int have, b, tile;
};

template <int NQ>
__device__ __forceinline__ TaPlace ta_find(const TaPlan& S, int x)
{
    const amp_attention_args& P = S.P;
    const int group = S.group, lane = threadIdx.x & 31;
    auto tiles = [&](int rows) { return rows <= S.split_rows ? 0 : (rows + ta_rows<NQ> - 1) / ta_rows<NQ>; };
    TaPlace f = {};
    if (!P.cu)
    {
        f.b = S.by_tiles.of(x);
        f.tile = x - f.b * tiles(S.each * group);
        f.have = 1;
        f.s = at_seq(P, f.b, S.each);
        return f;
    }
    // four sequences per lane at a time
    constexpr int EACH = 4;
    for (int b0 = 0; b0 < P.seqs; b0 += 32 * EACH)
    {
        int n[EACH], mine = 0;
        #pragma unroll
        for (int i = 0; i < EACH; ++i)
        {
            const int b = b0 + lane * EACH + i;
            n[i] = b < P.seqs ? tiles(at_count(P, b) * group) : 0;
            mine += n[i];
        }
        int sum = mine;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += y; }
        const uint32_t hit = __ballot_sync(0xffffffffu, x < sum);
        if (hit)
        {
            const int l = __ffs(hit) - 1;
            int left = x - (sum - mine), at = 0;             // (of lane l)
            #pragma unroll
            for (int i = 0; i < EACH - 1; ++i) if (at == i && left >= n[i]) { left -= n[i]; ++at; }
            f.have = 1;
            f.b = __shfl_sync(0xffffffffu, b0 + lane * EACH + at, l);
            f.tile = __shfl_sync(0xffffffffu, left, l);
            f.s = at_seq(P, f.b, 0);
            return f;
        }
        x -= __shfl_sync(0xffffffffu, sum, 31);
    }
    return f;
}

// A tile of values loses what has no finite magnitude, of keys that not all rows see, [0, from) and [to, count). By one warp, the one that
// multiplies: it has nothing to do while the weights are made, and its loop bears another branch: 8192 tokens 495 -> 497 us, six
// prompts of 390 tokens in windows of 128 32.3 -> 32.8 (the same work in the loading warps' loop: 4 to 26 us, and 2.5). Whether there was any.
template <typename T, int D, int KB>
__device__ __forceinline__ bool ta_sift(uint32_t at, int from, int to, int count)
{
    constexpr int CH = D / 8, PER = CH >= 32 ? 1 : 32 / CH, COPIES = KB / PER, BATCH = 4;
    const int lane = threadIdx.x & 31, r_lane = CH >= 32 ? 0 : lane / CH, c_lane = lane % CH;
    at += (c_lane >> 3) * (KB * 128);
    auto place = [&](int r) { return at + r * 128 + (((c_lane & 7) ^ (r & 7)) << 4); };
    // (of a tile that begins or ends among the keys that all rows see, only the other end)
    const int first = from <= 0 && to > 0 ? to / PER : 0, end = from > 0 && to >= KB ? min(from, count) : count, last = min(COPIES, (end + PER - 1) / PER);
    uint32_t odd = 0;
    #pragma unroll 1
    for (int i = first; i < last; i += BATCH)
    {
        uint4 v[BATCH];
        #pragma unroll
        for (int a = 0; a < BATCH; ++a) v[a] = at_lds16(place(min(i + a, last - 1) * PER + r_lane));
        #pragma unroll
        for (int a = 0; a < BATCH; ++a) odd |= at_odd<T>(v[a]);
    }
    if (!__any_sync(0xffffffffu, odd)) return false;
    #pragma unroll 1
    for (int i = first; i < last; ++i)
    {
        const int r = i * PER + r_lane;
        const uint4 v = at_lds16(place(r));
        if (at_odd<T>(v) && (r < from || r >= to)) at_sts16_even<T>(place(r), v);
    }
    ta_fence_async();
    __syncwarp();
    return true;
}

template <typename T, int D, int NQ>
__global__ __launch_bounds__(ta_threads<NQ>, (ta_ctas<D, NQ>))
void attention_tc_kernel(const TaPlan S)
{
    const amp_attention_args& P = S.P;
    constexpr int KB = ta_kb<NQ>, ST = ta_stages<D, NQ>, ROWS = ta_rows<NQ>;
    constexpr int Q_BYTES = 128 * D * 2, KV_BYTES = KB * D * 2, CH = D / 8;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    constexpr float TOP = BF ? 0.0f : AtType<T>::weight_top - TA_SLACK;      // (a maximum that has not moved yet lies up to the slack below)
    // tensor memory: S (two tiles or two buffers), then O
    constexpr int S_STEP = KB, O_COL = 2 * KB, TMEM = O_COL + NQ * (NQ == 2 ? 128 : D) <= 256 ? 256 : 512;
    static_assert(O_COL + (NQ == 2 ? 128 + D : D) <= TMEM && TMEM * ta_ctas<D, NQ> <= 512, "tensor memory");
    constexpr uint32_t IDESC_QK = ta_idesc(KB, BF, false), IDESC_PV = ta_idesc(D, BF, true);
    extern __shared__ __align__(1024) unsigned char ta_mem[];
    __shared__ uint64_t q_full, kv_full[ST], kv_free[ST], s_full[2], p_full[4], pv_done, o_full, end;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_odd;             // values without a finite magnitude were taken out of tiles that some rows see in part
    __shared__ TaPlace s_place;

    const int t = threadIdx.x, lane = t & 31, warp = __shfl_sync(0xffffffffu, t >> 5, 0);
    const int group = S.group;
    // (before tensor memory is taken: a CTA in front may still have to take its own here; those behind are let in when it is taken)
    if (S.pdl) pdl_wait();
    const int hx = S.by_kv.of(blockIdx.x), h = blockIdx.x - hx * P.kv_heads, from_last = S.by_slices.of(hx), slice = hx - from_last * S.slices;
    const int x = S.tiles - 1 - from_last;     // (the last tiles see most keys: first)
    if (warp == 0)
    {
        const TaPlace f = ta_find<NQ>(S, x);
        if (lane == 0) s_place = f;
    }
    else if (warp == 4 * NQ)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&s_tmem)), "r"((uint32_t) TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    else if (warp == 1 && lane == 0)
    {
        s_odd = 0;
        mbar_init(&q_full, 128 * NQ);
        for (int i = 0; i < ST; ++i) { mbar_init(&kv_full[i], TA_LOADERS); mbar_init(&kv_free[i], 1); }
        for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1);
        for (int i = 0; i < 4; ++i) mbar_init(&p_full[i], 128);
        mbar_init(&pv_done, 1);
        mbar_init(&o_full, 2);                 // the MMAs, and the warp that issues them (for s_odd)
        mbar_init(&end, 1);
        fence_mbar_init();
    }
    ta_fence_before();
    __syncthreads();
    ta_fence_after();
    const uint32_t tmem = s_tmem;
    if (S.pdl) pdl_launch_dependents();
    if (!s_place.have)
    {
        if (warp == 4 * NQ) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"((uint32_t) TMEM) : "memory");
        return;
    }
    const AtSeq seq = s_place.s;
    const int row0 = s_place.tile * ROWS, tok0 = S.by_group.of(row0), tok1 = min(S.by_group.of(row0 + ROWS - 1), seq.count - 1);
    const AtKeys keys = at_keys(P, seq.first + tok0, tok1 - tok0 + 1);
    const int n_all = (keys.count() + KB - 1) / KB;
    // (2^24 tiles of keys and 256 slices at most: the products are below 2^32)
    const int j0 = slice == 0 ? 0 : (int) ((unsigned) n_all * (unsigned) slice / (unsigned) S.slices);
    const int n = (slice + 1 == S.slices ? n_all : (int) ((unsigned) n_all * (unsigned) (slice + 1) / (unsigned) S.slices)) - j0;
    const uint32_t q_s = smem_u32(ta_mem), kv_s = q_s + NQ * Q_BYTES;
    const uint32_t full_s = smem_u32(&kv_full[0]), free_s = smem_u32(&kv_free[0]), sf = smem_u32(&s_full[0]), pf = smem_u32(&p_full[0]);
    const bool aligned = (q_s & 1023) == 0;    // (the swizzle needs the alignment that the declaration asks for)

    bool ok = aligned;
    if (!aligned && t == 0) atomicExch(&g_at_status, 2);
    // (a warp agrees on whether a wait was lost: what follows is done by whole warps)
    auto wait = [&](uint32_t bar, uint32_t parity)
    {
        if (ok && !__all_sync(0xffffffffu, ta_wait(bar, parity))) { ok = false; atomicExch(&g_at_status, 1); }
        return ok;
    };
    // registers of the block's launch (168 for each of its three warpgroups), given to those that hold rows
    if constexpr (NQ == 2)
    {
        if (warp < 4 * NQ) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;" ::: "memory");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 72;" ::: "memory");
    }

    if (warp < 4 * NQ)
    {
        // ---- softmax: thread t has row t of the CTA's ROWS ------------------------------------------------------------------
        const int i = warp >> 2;               // row tile
        const int row = row0 + t, tok = S.by_group.of(row), head = h * group + row - tok * group;
        const bool have = tok < seq.count;
        const int p = seq.first + tok;
        {
            // its row of Q, with the sign of the scale (the rest counts with |scale|; scale 0: scores of 0)
            const T* q = reinterpret_cast<const T*>(P.q) + (long long) (seq.row0 + tok) * P.q_token + (long long) head * P.q_head;
            const uint32_t flip = P.scale < 0.0f ? 0x80008000u : 0u;
            #pragma unroll 8
            for (int c = 0; c < CH; ++c)
            {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (have && P.scale != 0.0f) v = *reinterpret_cast<const uint4*>(q + c * 8);
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                             :: "r"(q_s + i * Q_BYTES + (c >> 3) * (128 * 128) + (t & 127) * 128 + (((c & 7) ^ (t & 7)) << 4)),
                                "r"(v.x ^ flip), "r"(v.y ^ flip), "r"(v.z ^ flip), "r"(v.w ^ flip) : "memory");
            }
            ta_fence_async();
            ta_arrive(smem_u32(&q_full));
        }
        // what its row sees of the keys, and a run of them that all rows of the row tile see: there no single key is looked at
        int n0, c1, len, from, to;
        at_row_keys(P, keys, p, n0, c1, len);
        at_whole_keys(P, keys, seq.first + S.by_group.of(row0 + 128 * i), seq.first + min(S.by_group.of(row0 + 128 * i + 127), seq.count - 1), from, to);

        const float sc = P.scale == 0.0f ? 1.0f : fabsf(S.scale2);
        const uint32_t lane_base = tmem + ((uint32_t) (32 * (warp & 3)) << 16);
        const uint32_t o_t = lane_base + O_COL + (NQ == 2 ? i * 128 : 0);
        float m = -INFINITY;
        f32x2 l2 = pack_f32x2(0.0f, 0.0f);
        float l = 0.0f;
        for (int j = 0; j < n; ++j)
        {
            const int buf = NQ == 2 ? i : (j & 1);
            if (!wait(sf + 8 * buf, (NQ == 2 ? j : j >> 1) & 1)) break;
            ta_fence_after();
            const uint32_t s_t = lane_base + buf * S_STEP;
            uint32_t s[KB];
            const int k0 = (j0 + j) * KB;
            const bool look = k0 < from || k0 + KB > to;
            float top4[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
            #pragma unroll
            for (int c = 0; c < KB / 2; c += 32) ta_ld32(s_t + c, s + c);
            ta_wait_ld();
            #pragma unroll
            for (int half = 0; half < 2; ++half)
            {
                // (the second half is on its way while the first one's maximum is taken)
                if (half == 0)
                {
                    #pragma unroll
                    for (int c = KB / 2; c < KB; c += 32) ta_ld32(s_t + c, s + c);
                }
                else ta_wait_ld();
                if (look)
                {
                    #pragma unroll
                    for (int c = half * (KB / 2); c < (half + 1) * (KB / 2); ++c)
                    {
                        const int at = k0 + c;
                        const bool see = at < n0 || (uint32_t) (at - c1) <= (uint32_t) len;
                        s[c] = see ? s[c] : 0xff800000u;
                    }
                }
                #pragma unroll
                for (int c = half * (KB / 2); c < (half + 1) * (KB / 2); c += 8)
                {
                    #pragma unroll
                    for (int e = 0; e < 4; ++e) top4[e] = fmaxf(fmaxf(top4[e], __uint_as_float(s[c + e])), __uint_as_float(s[c + 4 + e]));
                }
            }
            const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
            const bool move = top > m && (m == -INFINITY || (top - m) * sc > TA_SLACK);
            if (__any_sync(0xffffffffu, move))
            {
                const float f = move ? at_exp2((m - top) * sc) : 1.0f;       // (m of -inf: 0)
                if (move) m = top;
                l2 = mul_f32x2(l2, pack_f32x2(f, f));
                if (j > 0)
                {
                    constexpr int PIECE = NQ == 2 ? 32 : 16;             // columns at a time: 16 where two CTAs share the registers
                    // (one tile: S(j) was made before P V(j - 1), behind P V(j - 2): the phase is this one or the one in front)
                    if constexpr (NQ == 1) { if (!wait(smem_u32(&pv_done), (j - 1) & 1)) break; ta_fence_after(); }
                    #pragma unroll
                    for (int c = 0; c < D; c += PIECE)
                    {
                        uint32_t o[PIECE];
                        if constexpr (PIECE == 32) ta_ld32(o_t + c, o);
                        else ta_ld16(o_t + c, o);
                        ta_wait_ld();
                        #pragma unroll
                        for (int e = 0; e < PIECE; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        if constexpr (PIECE == 32) ta_st32(o_t + c, o);
                        else ta_st16(o_t + c, o);
                    }
                }
            }
            // 2^(s sc - m sc) in one step; where m sc is so large that its own rounding counts, the difference is taken first
            float by = sc, base = m == -INFINITY ? 0.0f : TOP - m * sc;
            if (__any_sync(0xffffffffu, fabsf(base) > TA_FAR))
            {
                const float at = m == -INFINITY ? 0.0f : -m;
                #pragma unroll
                for (int c = 0; c < KB; c += 2)
                {
                    const float2 d = unpack_f32x2(mul_f32x2(add_f32x2(pack_f32x2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), pack_f32x2(at, at)), pack_f32x2(sc, sc)));
                    s[c] = __float_as_uint(d.x);
                    s[c + 1] = __float_as_uint(d.y);
                }
                by = 1.0f;
                base = TOP;
            }
            const f32x2 sc2 = pack_f32x2(by, by), base2 = pack_f32x2(base, base);
            f32x2 sum2 = pack_f32x2(0.0f, 0.0f);             // (by itself: small weights beside a large l are lost one by one)
            #pragma unroll
            for (int half = 0; half < 2; ++half)
            {
                // (the MMAs over the first half's keys run while the second half is made)
                uint32_t w[KB / 4];
                #pragma unroll
                for (int e = 0; e < KB / 2; e += 2)
                {
                    const int c = half * (KB / 2) + e;
                    const f32x2 y = fma_f32x2(pack_f32x2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sc2, base2);
                    float2 x;
                    if ((e / 2) % 4 < ta_poly<D>) x = ta_exp2_pair(y);
                    else { x = unpack_f32x2(y); x.x = at_exp2(x.x); x.y = at_exp2(x.y); }
                    sum2 = add_f32x2(sum2, pack_f32x2(x.x, x.y));
                    w[e / 2] = AtType<T>::pack(x.x, x.y);
                }
                if constexpr (KB == 128) ta_st32(s_t + half * 32, w);
                else ta_st16(s_t + half * 16, w);
                ta_wait_st();
                ta_fence_before();
                ta_arrive(pf + 8 * (2 * buf + half));
            }
            l2 = add_f32x2(l2, sum2);
        }
        const float2 ls = unpack_f32x2(l2);
        l = ls.x + ls.y;
        if (n > 0 && ok)
        {
            wait(smem_u32(&o_full), 0);
            ta_fence_after();
        }
        // columns to which such values are added: infinity, minus infinity (both: NaN)
        uint32_t up[D / 32] = {}, down[D / 32] = {};
        const bool odd = s_odd;
        if (odd)
        {
            int whole_from, whole_to;          // (as the warp that multiplies has them)
            at_whole_keys(P, keys, seq.first + tok0, seq.first + tok1, whole_from, whole_to);
            const int end = min((j0 + n) * KB, keys.count());
            #pragma unroll 1
            for (int c = j0 * KB; c < end; ++c)
            {
                if (c >= whole_from && c < whole_to) { c = whole_to - 1; continue; }
                if (!have || !(c < n0 || (uint32_t) (c - c1) <= (uint32_t) len)) continue;
                const int key = keys.key(c), pg = S.g.page_of(key), page = P.table[(long long) s_place.b * P.table_row + pg];
                if ((unsigned) page >= (unsigned) P.pages) continue;
                const uint4* const v = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(P.v_cache) + h * P.v_head * 2
                                       + (unsigned long long) (page * S.g.v_page + (key - pg * P.page_size) * S.g.v_row) * 16);
                #pragma unroll
                for (int i = 0; i < D / 32; ++i)
                {
                    #pragma unroll 1
                    for (int e = 0; e < 4; ++e)
                    {
                        const uint4 x = v[4 * i + e];
                        if (!at_odd<T>(x)) continue;
                        const uint32_t y[4] = { x.x, x.y, x.z, x.w };
                        #pragma unroll
                        for (int k = 0; k < 4; ++k)
                        {
                            const float2 z = AtType<T>::unpack(y[k]);
                            const uint32_t is = AtType<T>::odd(y[k]), first = (is >> 15 & 1u) << (8 * e + 2 * k), second = (is >> 31) << (8 * e + 2 * k + 1);
                            up[i] |= (z.x < 0.0f ? 0 : first) | (z.y < 0.0f ? 0 : second);
                            down[i] |= (z.x > 0.0f ? 0 : first) | (z.y > 0.0f ? 0 : second);
                        }
                    }
                }
            }
            __syncwarp();
        }
        auto mend = [&](int i, uint32_t* o)
        {
            if (!odd) return;
            #pragma unroll
            for (int e = 0; e < 32; ++e)
                o[e] = __float_as_uint(__uint_as_float(o[e]) + (up[i] >> e & 1 ? INFINITY : 0.0f) + (down[i] >> e & 1 ? -INFINITY : 0.0f));
        };
        const float m2 = m == -INFINITY ? m : m * sc - TOP;  // (what the sums count from)
        if (S.slices > 1)
        {
            // a part: rows side by side, so that a warp writes whole lines; lost: NaN
            float* const part = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(P.workspace) + S.part_offset)
                                + (size_t) ((x * P.kv_heads + h) * S.slices + slice) * ta_part_floats(ROWS, D);
            if (n > 0)
            {
                #pragma unroll
                for (int c = 0; c < D; c += 32)
                {
                    uint32_t o[32];
                    ta_ld32(o_t + c, o);
                    ta_wait_ld();
                    mend(c / 32, o);
                    if (have)
                    {
                        #pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            reinterpret_cast<uint4*>(part)[((c + e) / 4) * ROWS + t] = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
            }
            if (have) reinterpret_cast<float2*>(part + ROWS * D)[t] = make_float2(m2, ok ? l : NAN);
        }
        else if (ok)
        {
            const float f = at_factor(P, p, l);
            #pragma unroll
            for (int c = 0; c < D; c += 32)
            {
                uint32_t o[32];
                if (n > 0) { ta_ld32(o_t + c, o); ta_wait_ld(); mend(c / 32, o); }
                if (have)
                {
                    #pragma unroll
                    for (int e = 0; e < 32; e += 8)
                    {
                        const float4 a = n > 0 ? make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3])) : make_float4(0, 0, 0, 0);
                        const float4 b = n > 0 ? make_float4(__uint_as_float(o[e + 4]), __uint_as_float(o[e + 5]), __uint_as_float(o[e + 6]), __uint_as_float(o[e + 7])) : make_float4(0, 0, 0, 0);
                        at_store8<T>(P, seq, tok, head, c + e, a, b, f, m2, l);
                    }
                }
            }
        }
    }
    else if (warp == 4 * NQ)
    {
        // ---- MMAs ------------------------------------------------------------------------------------------------------------
        int stage = 0; uint32_t wrap = 0;      // of the next tile in the order K0, K1, V0, K2, V1, ...
        auto next = [&]() { if (++stage == ST) { stage = 0; wrap ^= 1; } };
        auto qk = [&](int buf, int tile, int at)
        {
            const uint64_t a = ta_desc(q_s + tile * Q_BYTES, 0), b = ta_desc(kv_s + at * KV_BYTES, 0);
            if (ta_elect())
            {
                #pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    ta_mma_ss(tmem + buf * S_STEP, a + (kk >> 2) * (128 * 128 >> 4) + (kk & 3) * 2, b + (kk >> 2) * (KB * 128 >> 4) + (kk & 3) * 2, IDESC_QK, kk > 0);
                ta_commit(sf + 8 * buf);
            }
            __syncwarp();
        };
        auto pv = [&](int buf, int tile, int at, int half, bool first)
        {
            const uint64_t b = ta_desc(kv_s + at * KV_BYTES, KB * 128);
            if (ta_elect())
            {
                #pragma unroll
                for (int kk = half * (KB / 32); kk < (half + 1) * (KB / 32); ++kk)
                    ta_mma_ts(tmem + O_COL + (NQ == 2 ? tile * 128 : 0), tmem + buf * S_STEP + 8 * kk, b + kk * (16 * 128 >> 4), IDESC_PV, !first || kk > 0);
            }
            __syncwarp();
        };
        int whole_from, whole_to;              // keys that all rows of the CTA see
        at_whole_keys(P, keys, seq.first + tok0, seq.first + tok1, whole_from, whole_to);
        const int count = keys.count();
        auto commit = [&](uint32_t bar) { if (ta_elect()) ta_commit(bar); __syncwarp(); };
        if (n > 0 && wait(smem_u32(&q_full), 0) && wait(full_s + 8 * stage, wrap))
        {
            ta_fence_after();
            #pragma unroll
            for (int i = 0; i < NQ; ++i) qk(i, i, stage);
            commit(free_s + 8 * stage);
            next();
            for (int j = 0; j < n; ++j)
            {
                int kst = 0;
                if (j + 1 < n)
                {
                    if (!wait(full_s + 8 * stage, wrap)) break;
                    kst = stage;
                    next();
                }
                if constexpr (NQ == 1)
                {
                    if (j + 1 < n) { ta_fence_after(); qk((j + 1) & 1, 0, kst); commit(free_s + 8 * kst); }
                }
                if (!wait(full_s + 8 * stage, wrap)) break;
                const int vst = stage;
                next();
                const int k0 = (j0 + j) * KB;
                if ((k0 < whole_from || min(k0 + KB, count) > whole_to) && ta_sift<T, D, KB>(kv_s + vst * KV_BYTES, whole_from - k0, whole_to - k0, count - k0))
                    s_odd = 1;
                #pragma unroll
                for (int i = 0; i < NQ; ++i)
                {
                    const int buf = NQ == 2 ? i : (j & 1);
                    #pragma unroll
                    for (int half = 0; half < 2; ++half)
                    {
                        if (!wait(pf + 8 * (2 * buf + half), (NQ == 2 ? j : j >> 1) & 1)) break;
                        ta_fence_after();
                        pv(buf, i, vst, half, j == 0);
                    }
                    if (!ok) break;
                    if (i == NQ - 1) commit(free_s + 8 * vst);
                    if constexpr (NQ == 1) commit(smem_u32(&pv_done));
                    else if (j + 1 < n)
                    {
                        qk(i, i, kst);
                        if (i == NQ - 1) commit(free_s + 8 * kst);
                    }
                }
                if (!ok) break;
            }
            // (the end of the MMAs does not say that what the warp itself wrote is visible: its own arrival does)
            if (ok) { commit(smem_u32(&o_full)); if (lane == 0) ta_arrive(smem_u32(&o_full)); }
        }
        commit(smem_u32(&end));
        ta_wait(smem_u32(&end), 0);            // (bounded; the accumulators are given back only then)
    }
    else
    {
        // ---- keys and values, three warps: warp w makes every third of the copies of 32 x 16 bytes that a tile takes ---------------
        constexpr int PER = CH >= 32 ? 1 : 32 / CH, COPIES = KB / PER, MINE = (COPIES + TA_LOADERS - 1) / TA_LOADERS, LOOKS = (MINE * PER + 31) / 32;
        const int w = warp - 4 * NQ - 1, r_lane = CH >= 32 ? 0 : lane / CH, c_lane = lane % CH, count = keys.count();
        const unsigned char* const k_base = reinterpret_cast<const unsigned char*>(P.k_cache) + h * P.k_head * 2 + c_lane * 16;
        const unsigned char* const v_base = reinterpret_cast<const unsigned char*>(P.v_cache) + h * P.v_head * 2 + c_lane * 16;
        const int* const table = P.table + (long long) s_place.b * P.table_row;
        // lane l looks up the l-th, (l + 32)-th ... of the warp's rows: page and row in it
        struct Rows { int page[LOOKS], row[LOOKS]; };        // (row -1: behind the last key, -2: no row of this warp)
        auto look_up = [&](int j, Rows& x)
        {
            #pragma unroll
            for (int g = 0; g < LOOKS; ++g)
            {
                const int q = lane + 32 * g, r = (w + TA_LOADERS * (q / PER)) * PER + q % PER, c = (j0 + j) * KB + r;
                x.page[g] = -1;
                x.row[g] = q < MINE * PER && r < KB ? (c < count ? 0 : -1) : -2;
                if (x.row[g] == 0)
                {
                    const int key = keys.key(c), pg = S.g.page_of(key);
                    x.page[g] = table[pg];
                    x.row[g] = key - pg * P.page_size;
                }
            }
        };
        int issued = 0, stage = 0;
        auto hand_over = [&](int tile)
        {
            ta_fence_async();
            __syncwarp();
            if (lane == 0) ta_arrive(full_s + 8 * (tile % ST));
        };
        auto copy_tile = [&](const Rows& x, bool is_v)
        {
            uint32_t off[LOOKS], have = 0xffffffffu;         // offsets in pieces of 16 bytes; lanes whose rows are all there
            int state[LOOKS];                                // 1: there, 0: behind the last key, -1: on a page outside the pool
            #pragma unroll
            for (int g = 0; g < LOOKS; ++g)
            {
                state[g] = x.row[g] == -2 ? 1 : x.row[g] == -1 ? 0 : (unsigned) x.page[g] < (unsigned) P.pages ? 1 : -1;
                off[g] = x.row[g] < 0 || state[g] < 0 ? 0 : is_v ? x.page[g] * S.g.v_page + x.row[g] * S.g.v_row : x.page[g] * S.g.k_page + x.row[g] * S.g.k_row;
                have &= __ballot_sync(0xffffffffu, state[g] > 0);
            }
            if (issued >= ST && !wait(free_s + 8 * stage, (issued / ST - 1) & 1)) return;
            const unsigned char* const base = is_v ? v_base : k_base;
            const uint32_t to = kv_s + stage * KV_BYTES + (c_lane >> 3) * (KB * 128);
            if (have == 0xffffffffu)
            {
                #pragma unroll
                for (int i = 0; i < MINE; ++i)
                {
                    const int r = (w + TA_LOADERS * i) * PER + r_lane;
                    const uint32_t o = __shfl_sync(0xffffffffu, off[i * PER / 32], i * PER % 32 + r_lane);
                    if (COPIES % TA_LOADERS == 0 || i + 1 < MINE || w + TA_LOADERS * i < COPIES)
                        cp_async16_s(to + r * 128 + (((c_lane & 7) ^ (r & 7)) << 4), base + (unsigned long long) o * 16);
                }
            }
            else
            {
                #pragma unroll 1
                for (int i = 0; i < MINE; ++i)
                {
                    const int r = (w + TA_LOADERS * i) * PER + r_lane, from = (i * PER) % 32 + r_lane;
                    uint32_t o = 0;
                    int st = 0;
                    #pragma unroll
                    for (int g = 0; g < LOOKS; ++g)
                    {
                        const uint32_t y = __shfl_sync(0xffffffffu, off[g], from);
                        const int z = __shfl_sync(0xffffffffu, state[g], from);
                        if (g == i * PER / 32) { o = y; st = z; }
                    }
                    const uint32_t dst = to + r * 128 + (((c_lane & 7) ^ (r & 7)) << 4);
                    if (w + TA_LOADERS * i < COPIES)
                    {
                        // a key that cannot be found is NaN to the rows that see it, its value 0; zeros behind the last key
                        if (st < 0 && !is_v) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" :: "r"(dst), "r"(0x7fff7fffu) : "memory");
                        else at_copy16(dst, st > 0 ? base + (unsigned long long) o * 16 : base, st > 0);
                    }
                }
            }
            cp_async_commit();
            if (issued >= TA_AHEAD) { asm volatile("cp.async.wait_group %0;" :: "n"(TA_AHEAD) : "memory"); hand_over(issued - TA_AHEAD); }
            ++issued;
            stage = stage + 1 == ST ? 0 : stage + 1;
        };
        // K0, then K1, V0, K2, V1, ...: a tile's rows are looked up two tiles ahead, and kept from its keys to its values
        Rows now, next, then;
        if (n > 0)
        {
            look_up(0, now);
            if (n > 1) look_up(1, next);
            copy_tile(now, false);
            #pragma unroll 1
            for (int j = 0; j < n && ok; ++j)
            {
                if (j + 1 < n) copy_tile(next, false);
                if (!ok) break;
                if (j + 2 < n) look_up(j + 2, then);
                copy_tile(now, true);
                now = next;
                next = then;
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (ok) for (int tile = max(0, issued - TA_AHEAD); tile < issued; ++tile) hand_over(tile);
    }
    ta_fence_before();
    __syncthreads();
    if (warp == 4 * NQ)
    {
        ta_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"((uint32_t) TMEM) : "memory");
    }
}

// Joins the slices of row tile x of key-value head h (blockIdx.x), 16 values of every row (blockIdx.y)
template <typename T, int D, int NQ>
__global__ __launch_bounds__(128 * NQ)
void attention_tc_join_kernel(const TaPlan S)
{
    const amp_attention_args& P = S.P;
    constexpr int ROWS = ta_rows<NQ>;
    __shared__ TaPlace s_place;
    const int t = threadIdx.x, x = S.by_kv.of(blockIdx.x), h = blockIdx.x - x * P.kv_heads, group = S.group;
    if (S.pdl) { pdl_wait(); pdl_launch_dependents(); }
    if (t < 32)
    {
        const TaPlace f = ta_find<NQ>(S, x);
        if (t == 0) s_place = f;
    }
    __syncthreads();
    if (!s_place.have) return;
    const AtSeq seq = s_place.s;
    const int row = s_place.tile * ROWS + t, tok = S.by_group.of(row);
    if (tok >= seq.count) return;
    const float* const parts = reinterpret_cast<const float*>(reinterpret_cast<const unsigned char*>(P.workspace) + S.part_offset)
                               + (size_t) blockIdx.x * S.slices * ta_part_floats(ROWS, D);
    auto ml = [&](int i) { return reinterpret_cast<const float2*>(parts + i * ta_part_floats(ROWS, D) + ROWS * D)[t]; };
    float m = -INFINITY, l = 0.0f;
    for (int i = 0; i < S.slices; ++i) m = fmaxf(m, ml(i).x);
    const float base = m == -INFINITY ? 0.0f : m;
    float4 o[4];
    #pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    #pragma unroll 2
    for (int i = 0; i < S.slices; ++i)
    {
        const float2 v = ml(i);
        if (v.y == 0.0f) continue;             // (a slice without keys wrote nothing else)
        const float f = at_exp2(v.x - base);
        l += v.y != v.y ? v.y : v.y * f;
        const float4* p = reinterpret_cast<const float4*>(parts + i * ta_part_floats(ROWS, D)) + (size_t) blockIdx.y * 4 * ROWS + t;
        #pragma unroll
        for (int c = 0; c < 4; ++c)
        {
            const float4 y = p[c * ROWS];
            o[c].x += y.x * f; o[c].y += y.y * f; o[c].z += y.z * f; o[c].w += y.w * f;
        }
    }
    const int head = h * group + row - tok * group;
    const float f = at_factor(P, seq.first + tok, l);
    at_store8<T>(P, seq, tok, head, blockIdx.y * 16, o[0], o[1], f, m, l);
    at_store8<T>(P, seq, tok, head, blockIdx.y * 16 + 8, o[2], o[3], f, m, l);
}

template <typename T, int D, int NQ>
static int ta_launch(const TaPlan& S, cudaStream_t stream)
{
    const amp_attention_args& P = S.P;
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return cuda_rc(e, "attention device");
    if (cudaError_t e = ensure_smem(attention_tc_kernel<T, D, NQ>, ta_smem<D, NQ>, dev)) return cuda_rc(e, "attention shared memory");
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(S.tiles * S.slices * P.kv_heads, 1, 1);
    cfg.blockDim = dim3(ta_threads<NQ>, 1, 1);
    cfg.dynamicSmemBytes = ta_smem<D, NQ>;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = S.pdl ? 1 : 0;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, attention_tc_kernel<T, D, NQ>, S)) return cuda_rc(e, "attention launch");
    if (S.slices == 1) return 0;
    cfg.gridDim = dim3(S.tiles * P.kv_heads, D / 16, 1);
    cfg.blockDim = dim3(128 * NQ, 1, 1);
    cfg.dynamicSmemBytes = 0;
    return cuda_rc(cudaLaunchKernelEx(&cfg, attention_tc_join_kernel<T, D, NQ>, S), "attention join launch");
}

template <typename T>
static int ta_launch_dim(const TaPlan& S, cudaStream_t stream)
{
    if (S.P.dim == 256) return ta_launch<T, 256, 1>(S, stream);
    if (S.P.dim == 128) return S.nq == 1 ? ta_launch<T, 128, 1>(S, stream) : ta_launch<T, 128, 2>(S, stream);
    return S.nq == 1 ? ta_launch<T, 64, 1>(S, stream) : ta_launch<T, 64, 2>(S, stream);
}

int attention_tc(TaPlan& S, cudaStream_t stream)
{
    const amp_attention_args& P = S.P;
    if (S.tiles == 0) return 0;
    const int tile = 128 * S.nq;
    S.group = P.heads / P.kv_heads; S.each = P.tokens / P.seqs;
    S.by_group = at_div(S.group); S.by_kv = at_div(P.kv_heads); S.by_slices = at_div(S.slices);
    S.by_tiles = at_div(P.cu ? 1 : ((long) S.each * S.group + tile - 1) / tile);
    return S.P.bf16 ? ta_launch_dim<__nv_bfloat16>(S, stream) : ta_launch_dim<__half>(S, stream);
}

// (read and cleared in one step: what another host thread's call sets meanwhile is kept for the next look)
__device__ int g_at_taken;
__global__ void attention_status_kernel() { g_at_taken = atomicExch(&g_at_status, 0); }

}  // namespace amp

AMP_API int amp_b200_attention_status(int* out)
{
    using namespace amp;
    static std::mutex one;                     // (one look at a time uses g_at_taken)
    std::lock_guard<std::mutex> lock(one);
    int v = 0;
    if (cudaError_t e = cudaDeviceSynchronize()) return cuda_rc(e, "status wait");       // (streams that do not wait for the default one, too)
    attention_status_kernel<<<1, 1>>>();
    if (cudaError_t e = cudaGetLastError()) return cuda_rc(e, "status read");
    if (cudaError_t e = cudaMemcpyFromSymbol(&v, g_at_taken, sizeof(int))) return cuda_rc(e, "status read");
    if (out) *out = v;
    return 0;
}
