// Attention of a few new tokens per sequence over a paged key-value cache: one pass over the keys and values, split over the
// cache's length and joined.
//
// The query heads that share a key-value head, times the sequence's new tokens, are the rows of one problem (row = token * group +
// head); 16 rows make a row tile, the M of mma.sync m16n8k16. The keys that a sequence's new tokens see, counted through (the
// first tokens and the window's without what lies between), are cut into units of 64. All units of the call, ordered (sequence,
// head, row tile, unit), are cut into equal contiguous ranges, one per CTA: the lengths stand on the device, so that a captured
// graph replays with other lengths, and long and short sequences share the device evenly. What a CTA holds of a (sequence, head,
// row tile) that other CTAs share goes to the workspace as partial result (o, m, l); a second kernel joins them in ascending key
// order, so that the sums are the same in every run.
//
// A warp owns 16 keys of every unit and a ring of stages of its own, filled with 16-byte asynchronous copies by its own lanes: the
// loop has no barrier between warps, each keeps its own m, l and o, and the four meet when a segment ends. The rings run ahead over
// the ends of segments.
#include "attention_tc.cuh"

namespace amp {

constexpr int AT_ROWS = 16;                    // rows of a row tile
constexpr int AT_UNIT = 64;                    // keys of a unit: 16 per warp
constexpr int AT_DESC = 8;                     // ints of a CTA's description for the join

template <int D> constexpr int at_stages = D == 64 ? 4 : 3;
template <int D> constexpr int at_ctas = D == 64 ? 3 : (D == 128 ? 2 : 1);     // per SM
template <int D> constexpr int at_stage_bytes = 64 * D;        // of one warp: 16 keys and 16 values; also 16 x D floats of o
template <int D> constexpr int at_smem = 4 * at_stages<D> * at_stage_bytes<D>;

struct AtPlan
{
    amp_attention_args P;
    int grid;                                  // CTAs of the split form
    int split_rows;                            // with cu: sequences of more rows (tokens x group) are the prompt form's
    int whole;                                 // 1: every (sequence, head, row tile) belongs to one CTA, nothing to join
    int pdl;
    float scale2;                              // scale * log2(e)
};

__device__ __forceinline__ void at_ldsm4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void at_ldsm4_trans(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <typename T>
__device__ __forceinline__ void at_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Row tiles of a sequence, and units of each of them
__device__ __forceinline__ int at_row_tiles(const AtPlan& S, const AtSeq& s)
{
    const int rows = s.count * (S.P.heads / S.P.kv_heads);
    return rows > S.split_rows ? 0 : (rows + AT_ROWS - 1) / AT_ROWS;
}

__device__ __forceinline__ int at_units(const AtKeys& k) { return max(1, (k.count() + AT_UNIT - 1) / AT_UNIT); }

// A place in the order of units
struct AtCursor
{
    int b, h, rt, u, tiles, units;
    AtSeq s;
    AtKeys k;

    __device__ __forceinline__ void load(const AtPlan& S)
    {
        s = at_seq(S.P, b);
        k = at_keys(S.P, s.first, s.count);
        tiles = at_row_tiles(S, s);
        units = at_units(k);
    }
    // to the next unit; the caller knows that there is one
    __device__ __forceinline__ bool advance(const AtPlan& S)
    {
        if (++u < units) return false;
        u = 0;
        if (++rt < tiles) return true;
        rt = 0;
        if (++h < S.P.kv_heads) return true;
        h = 0;
        do { ++b; load(S); } while (!tiles && b + 1 < S.P.seqs);
        return true;
    }
};

// Workspace: descriptions of the CTAs' first segments, then two partial results per CTA (16 rows of o, their m and l): of the
// segment that began before the CTA, and of the one that it does not end
__host__ __device__ constexpr size_t at_desc_bytes(int grid) { return ((size_t) grid * AT_DESC * 4 + 127) / 128 * 128; }
__host__ __device__ constexpr size_t at_part_floats(int dim) { return (size_t) AT_ROWS * (dim + 2); }

template <typename T, int D>
__global__ __launch_bounds__(128, at_ctas<D>)
void attention_split_kernel(const AtPlan S)
{
    const amp_attention_args& P = S.P;
    constexpr int NST = at_stages<D>, STAGE = at_stage_bytes<D>, CHUNKS = D / 8;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float s_ml[4][AT_ROWS][2];
    __shared__ uint32_t s_flags[4][NST];       // per warp and stage: keys that count, keys on a page outside the pool (upper half)
    __shared__ long long s_scan[128];
    __shared__ int s_place[5];

    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, cta = blockIdx.x;
    const int group = P.heads / P.kv_heads;
    if (S.pdl) { pdl_wait(); pdl_launch_dependents(); }
    int* desc = reinterpret_cast<int*>(P.workspace) + (size_t) cta * AT_DESC;

    // the CTA's range of units
    AtCursor in;
    long long left;
    if (S.whole)
    {
        in.b = 0; in.load(S);                                // (all sequences have as many tokens)
        const int per = P.kv_heads * in.tiles;
        in.b = cta / per; in.h = cta % per / in.tiles; in.rt = cta % in.tiles; in.u = 0;
        in.load(S);
        left = in.units;
    }
    else
    {
        // prefix sums over the sequences: a thread counts a run of them
        const int run = (P.seqs + 127) / 128, b0 = min(P.seqs, t * run), b1 = min(P.seqs, b0 + run);
        long long mine = 0;
        for (int b = b0; b < b1; ++b)
        {
            const AtSeq s = at_seq(P, b);
            mine += (long long) P.kv_heads * at_row_tiles(S, s) * at_units(at_keys(P, s.first, s.count));
        }
        long long sum = mine;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const long long x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        if (lane == 31) s_scan[warp] = sum;
        __syncthreads();
        long long total = 0;
        for (int w = 0; w < 4; ++w) { if (w == warp) sum += total; total += s_scan[w]; }
        const int ctas = (int) min((long long) S.grid, total);
        if (cta >= ctas)
        {
            if (t == 0) desc[0] = -1;
            return;
        }
        const long long u0 = cta * total / ctas;
        left = (cta + 1) * total / ctas - u0;
        if (u0 >= sum - mine && u0 < sum)                    // in this thread's run of sequences
        {
            long long at = u0 - (sum - mine);
            for (int b = b0; b < b1; ++b)
            {
                AtCursor c;
                c.b = b; c.load(S);
                const long long n = (long long) P.kv_heads * c.tiles * c.units;
                if (at < n)
                {
                    s_place[0] = b;
                    s_place[1] = (int) (at / (c.tiles * c.units));
                    s_place[2] = (int) (at / c.units) % c.tiles;
                    s_place[3] = (int) (at % c.units);
                    break;
                }
                at -= n;
            }
        }
        __syncthreads();
        in.b = s_place[0]; in.h = s_place[1]; in.rt = s_place[2]; in.u = s_place[3];
        in.load(S);
        if (t == 0)
        {
            // a segment that began before this CTA: which CTAs hold parts of it
            const long long g0 = u0 - in.u, g1 = g0 + in.units;
            desc[0] = in.u ? in.b : -1;
            desc[1] = in.h;
            desc[2] = in.rt;
            desc[3] = (int) (((g0 + 1) * ctas - 1) / total);
            desc[4] = (int) ((g1 * ctas - 1) / total);
        }
    }
    const bool began_before = in.u > 0;

    const uint32_t ring = smem_u32(smem) + warp * NST * STAGE;
    const T* const kc = reinterpret_cast<const T*>(P.k_cache);
    const T* const vc = reinterpret_cast<const T*>(P.v_cache);

    // ---- loads: lane l < 16 looks up key l of the warp's sixteen, the table entry a unit ahead -----------------------------
    AtCursor ld = in;
    long long to_load = left;
    int pre_page = 0, pre_row = 0;
    bool pre_live = false;
    auto look_up = [&]() {
        const int i = ld.u * AT_UNIT + warp * 16 + (lane & 15);
        pre_live = i < ld.k.count();
        if (pre_live)
        {
            const int j = ld.k.key(i), pg = j / P.page_size;
            pre_row = j - pg * P.page_size;
            pre_page = P.table[(long long) ld.b * P.table_row + pg];
        }
    };
    auto issue = [&](int stage) {
        if (to_load > 0)
        {
            const bool bad = pre_live && (pre_page < 0 || pre_page >= P.pages);
            const uint32_t live = __ballot_sync(0xffffffffu, pre_live) & 0xffffu, wrong = __ballot_sync(0xffffffffu, bad) & 0xffffu;
            if (lane == 0) s_flags[warp][stage] = live | (wrong << 16);
            const bool fetch = pre_live && !bad;
            const long long ko = fetch ? pre_page * P.k_page + pre_row * P.k_row + ld.h * P.k_head : 0;
            const long long vo = fetch ? pre_page * P.v_page + pre_row * P.v_row + ld.h * P.v_head : 0;
            const uint32_t have = live & ~wrong;
            const uint32_t at = ring + stage * STAGE;
            constexpr int PER = 32 / CHUNKS > 0 ? 32 / CHUNKS : 1;          // rows per warp-wide copy
            #pragma unroll
            for (int r0 = 0; r0 < 16; r0 += PER)
            {
                const int r = r0 + (CHUNKS >= 32 ? 0 : lane / CHUNKS), c = lane % CHUNKS;
                const long long k = __shfl_sync(0xffffffffu, ko, r), v = __shfl_sync(0xffffffffu, vo, r);
                const bool ok = (have >> r) & 1;
                const uint32_t off = r * (2 * D) + ((c ^ (r & 7)) << 4);
                at_copy16(at + off, kc + k + c * 8, ok);
                at_copy16(at + STAGE / 2 + off, vc + v + c * 8, ok);
            }
            if (--to_load > 0) { ld.advance(S); look_up(); }
        }
        cp_async_commit();
    };
    look_up();
    #pragma unroll
    for (int i = 0; i < NST; ++i) issue(i);

    // ---- the segments of the range -------------------------------------------------------------------------------------------
    uint32_t qf[D / 16][4];
    float o[D / 8][4], m[2], l[2];
    int p_row[2];                                            // positions of the lane's two rows
    bool fresh = true, first_segment = true;
    int stage = 0;
    while (left > 0)
    {
        if (fresh)
        {
            #pragma unroll
            for (int i = 0; i < 2; ++i)
            {
                const int r = in.rt * AT_ROWS + (lane >> 2) + 8 * i, tok = r / group;
                const bool have = tok < in.s.count;
                p_row[i] = in.s.first + tok;
                const T* q = reinterpret_cast<const T*>(P.q) + (long long) (in.s.row0 + tok) * P.q_token + (long long) (in.h * group + r - tok * group) * P.q_head + (lane & 3) * 2;
                #pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                {
                    qf[ks][i] = have ? *reinterpret_cast<const uint32_t*>(q + ks * 16) : 0u;
                    qf[ks][i + 2] = have ? *reinterpret_cast<const uint32_t*>(q + ks * 16 + 8) : 0u;
                }
                m[i] = -INFINITY;
                l[i] = 0.0f;
            }
            #pragma unroll
            for (int n = 0; n < D / 8; ++n) { o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f; }
            fresh = false;
        }
        cp_async_wait(NST - 1);
        __syncwarp();
        const uint32_t flags = s_flags[warp][stage];
        const uint32_t kb = ring + stage * STAGE, vb = kb + STAGE / 2;
        if (flags & 0xffffu)
        {
            // s = q k^T: rows x 16 keys, two n tiles
            float s[2][4] = {};
            #pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
            {
                const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * ks + ((lane >> 3) & 1);
                uint32_t f[4];
                at_ldsm4(kb + r * (2 * D) + ((c ^ (r & 7)) << 4), f);
                at_mma<T>(s[0], qf[ks], f[0], f[1]);
                at_mma<T>(s[1], qf[ks], f[2], f[3]);
            }
            float top[2] = { m[0], m[1] };
            const bool per_row = in.s.count > 1;
            #pragma unroll
            for (int n = 0; n < 2; ++n)
            {
                #pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    const int c = n * 8 + (lane & 3) * 2 + (e & 1);
                    bool see = (flags >> c) & 1;
                    if (per_row) see = see && at_sees(P, p_row[e >> 1], in.k.key(in.u * AT_UNIT + warp * 16 + c));
                    const float x = (flags >> (16 + c)) & 1 ? NAN : s[n][e] * S.scale2;
                    s[n][e] = see ? x : -INFINITY;
                    top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
                }
            }
            #pragma unroll
            for (int i = 0; i < 2; ++i)
            {
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
                top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
            }
            if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1]))
            {
                #pragma unroll
                for (int i = 0; i < 2; ++i)
                {
                    const float f = top[i] > m[i] ? exp2f(m[i] - top[i]) : 1.0f;
                    m[i] = top[i];
                    l[i] *= f;
                    #pragma unroll
                    for (int n = 0; n < D / 8; ++n) { o[n][2 * i] *= f; o[n][2 * i + 1] *= f; }
                }
            }
            const float base0 = m[0] == -INFINITY ? 0.0f : m[0], base1 = m[1] == -INFINITY ? 0.0f : m[1];
            #pragma unroll
            for (int n = 0; n < 2; ++n)
            {
                s[n][0] = exp2f(s[n][0] - base0); s[n][1] = exp2f(s[n][1] - base0);
                s[n][2] = exp2f(s[n][2] - base1); s[n][3] = exp2f(s[n][3] - base1);
                l[0] += s[n][0] + s[n][1];
                l[1] += s[n][2] + s[n][3];
            }
            const uint32_t pf[4] = { AtType<T>::pack(s[0][0], s[0][1]), AtType<T>::pack(s[0][2], s[0][3]),
                                     AtType<T>::pack(s[1][0], s[1][1]), AtType<T>::pack(s[1][2], s[1][3]) };
            #pragma unroll
            for (int n = 0; n < D / 16; ++n)
            {
                const int r = lane & 15, c = 2 * n + (lane >> 4);
                uint32_t f[4];
                at_ldsm4_trans(vb + r * (2 * D) + ((c ^ (r & 7)) << 4), f);
                at_mma<T>(o[2 * n], pf, f[0], f[1]);
                at_mma<T>(o[2 * n + 1], pf, f[2], f[3]);
            }
        }
        __syncwarp();
        --left;
        const bool ends = in.u + 1 == in.units;
        if (ends || left == 0)
        {
            // the four warps' parts meet in the stage each has just read
            #pragma unroll
            for (int i = 0; i < 2; ++i)
            {
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
                if ((lane & 3) == 0) { s_ml[warp][(lane >> 2) + 8 * i][0] = m[i]; s_ml[warp][(lane >> 2) + 8 * i][1] = l[i]; }
            }
            __syncthreads();
            #pragma unroll
            for (int i = 0; i < 2; ++i)
            {
                const int r = (lane >> 2) + 8 * i;
                const float top = fmaxf(fmaxf(s_ml[0][r][0], s_ml[1][r][0]), fmaxf(s_ml[2][r][0], s_ml[3][r][0]));
                const float f = m[i] == -INFINITY ? 0.0f : exp2f(m[i] - top);
                #pragma unroll
                for (int n = 0; n < D / 8; ++n)
                {
                    const int col = (n * 8 + (lane & 3) * 2) ^ ((r & 3) << 3);
                    asm volatile("st.shared.v2.f32 [%0], {%1, %2};" :: "r"(kb + (r * D + col) * 4), "f"(o[n][2 * i] * f), "f"(o[n][2 * i + 1] * f) : "memory");
                }
            }
            __syncthreads();
            const bool shared = !S.whole && ((first_segment && began_before) || !ends);
            const int slot = 2 * cta + (first_segment && began_before ? 0 : 1);
            float* const part = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(P.workspace) + at_desc_bytes(S.grid)) + slot * at_part_floats(D);
            for (int i = t; i < AT_ROWS * D / 4; i += 128)
            {
                const int r = i / (D / 4), c = (i % (D / 4)) * 4;
                const int row = in.rt * AT_ROWS + r, tok = row / group;
                if (tok >= in.s.count) break;                // (rows ascend with i)
                float top = -INFINITY, sum = 0.0f;
                #pragma unroll
                for (int w = 0; w < 4; ++w) top = fmaxf(top, s_ml[w][r][0]);
                #pragma unroll
                for (int w = 0; w < 4; ++w) sum += s_ml[w][r][0] == -INFINITY ? s_ml[w][r][1] : s_ml[w][r][1] * exp2f(s_ml[w][r][0] - top);
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                #pragma unroll
                for (int w = 0; w < 4; ++w)
                {
                    const float4 y = *reinterpret_cast<const float4*>(smem + (w * NST + stage) * STAGE + (r * D + (c ^ ((r & 3) << 3))) * 4);
                    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
                }
                if (shared)
                {
                    *reinterpret_cast<float4*>(part + r * D + c) = x;
                    if (c == 0) *reinterpret_cast<float2*>(part + AT_ROWS * D + 2 * r) = make_float2(top, sum);
                }
                else
                    at_store<T>(P, in.s, tok, in.h * group + row - tok * group, c, x, top, sum);
            }
            __syncthreads();
            fresh = true;
            first_segment = false;
        }
        issue(stage);
        stage = stage + 1 == NST ? 0 : stage + 1;
        if (left > 0) in.advance(S);
    }
}

// One CTA per CTA of the split form (x) and row of a row tile (y): joins the parts of the segment whose second part that CTA holds
template <typename T, int D>
__global__ __launch_bounds__(128)
void attention_join_kernel(const AtPlan S)
{
    const amp_attention_args& P = S.P;
    if (S.pdl) { pdl_wait(); pdl_launch_dependents(); }
    __shared__ float s_red[4], s_sum[4];
    __shared__ float4 s_o[4][D / 4];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, cta = blockIdx.x + 1, r = blockIdx.y;
    const int* desc = reinterpret_cast<const int*>(P.workspace) + (size_t) cta * AT_DESC;
    const int4 d = *reinterpret_cast<const int4*>(desc);
    if (d.x < 0 || d.w != cta - 1) return;
    const int last = desc[4], group = P.heads / P.kv_heads;
    const AtSeq s = at_seq(P, d.x);
    const int row = d.z * AT_ROWS + r, tok = row / group;
    if (tok >= s.count) return;
    const float* const parts = reinterpret_cast<const float*>(reinterpret_cast<const unsigned char*>(P.workspace) + at_desc_bytes(S.grid));
    // part i of the segment: the first is the end of its CTA's range, the others are the beginning of theirs
    const int n = last - d.w + 1;
    auto part = [&](int i) { return parts + (size_t) (2 * (d.w + i) + (i ? 0 : 1)) * at_part_floats(D); };

    float m = -INFINITY;
    for (int i = t; i < n; i += 128) m = fmaxf(m, part(i)[AT_ROWS * D + 2 * r]);
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s_red[warp] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    const float base = m == -INFINITY ? 0.0f : m;

    // a warp adds every fourth part up, a lane D / 32 values of the row (in pieces of four)
    constexpr int PIECES = D / 4, EACH = (PIECES + 31) / 32;
    float4 acc[EACH];
    #pragma unroll
    for (int e = 0; e < EACH; ++e) acc[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
    #pragma unroll 4
    for (int i = warp; i < n; i += 4)
    {
        const float* p = part(i);
        const float2 ml = *reinterpret_cast<const float2*>(p + AT_ROWS * D + 2 * r);
        const float f = exp2f(ml.x - base);
        l += ml.x == -INFINITY ? ml.y : ml.y * f;            // (an l of NaN stays one)
        #pragma unroll
        for (int e = 0; e < EACH; ++e)
        {
            const int c = lane + 32 * e;
            if (PIECES % 32 == 0 || c < PIECES)
            {
                const float4 x = reinterpret_cast<const float4*>(p + r * D)[c];
                acc[e].x += x.x * f; acc[e].y += x.y * f; acc[e].z += x.z * f; acc[e].w += x.w * f;
            }
        }
    }
    if (lane == 0) s_sum[warp] = l;
    #pragma unroll
    for (int e = 0; e < EACH; ++e) if (PIECES % 32 == 0 || lane + 32 * e < PIECES) s_o[warp][lane + 32 * e] = acc[e];
    __syncthreads();
    l = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
    for (int c = t; c < PIECES; c += 128)
    {
        float4 x = s_o[0][c];
        #pragma unroll
        for (int w = 1; w < 4; ++w) { const float4 y = s_o[w][c]; x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w; }
        at_store<T>(P, s, tok, d.y * group + row - tok * group, c * 4, x, m, l);
    }
}

struct AtDevice { int sms; };

static const AtDevice* at_device(int* rc)
{
    static AtDevice devices[64];
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) { *rc = cuda_rc(e, "attention device"); return nullptr; }
    if (dev < 0 || dev >= 64) { *rc = fail(AMP_E_UNSUPPORTED, "attention: device %d", dev); return nullptr; }
    if (!devices[dev].sms)
    {
        int n = 0;
        if (cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev)) { *rc = cuda_rc(e, "attention device"); return nullptr; }
        devices[dev].sms = n;
    }
    return &devices[dev];
}

// Sequences that fit into this many keys are not split: nothing is joined then
constexpr int AT_WHOLE_KEYS = 256;
// Rows (tokens x group) up to which a sequence takes the split form; beyond, the prompt form
constexpr int AT_SPLIT_ROWS = 32;

static int at_grid(int dim, int sms) { return sms * (dim == 64 ? at_ctas<64> : dim == 128 ? at_ctas<128> : at_ctas<256>); }

// How a call is cut up: by its sizes alone (the lengths are on the device)
struct AtCut
{
    bool split, tc;                            // forms that are launched
    int whole, grid;                           // split form
    int tiles, slices;                         // prompt form
    size_t tc_offset, bytes;                   // of the workspace
};

// Slices of the keys of each of `items` row tiles, `kt` key tiles long at most: waves of CTAs, each its share of the key tiles and a
// set-up of about two, and a join worth four
static int ta_slices(long items, long kt, int sms)
{
    int best = 1;
    double cost = 1e30;
    for (int s = 1; s <= kt && s * items <= 4l * sms && s <= 256; ++s)
    {
        const double c = (double) ((items * s + sms - 1) / sms) * ((double) ((kt + s - 1) / s) + 2) + (s > 1 ? 4 : 0);
        if (c < cost * 0.97) { cost = c; best = s; }
    }
    return best;
}

static AtCut at_cut(int tokens, int seqs, int heads, int kv_heads, int dim, bool ragged, long max_keys, int window, int sinks, int sms)
{
    AtCut C = {};
    const long group = heads / kv_heads, all = tokens * group, each = all / seqs;
    C.split = ragged || each <= AT_SPLIT_ROWS;
    C.tc = ragged ? all > AT_SPLIT_ROWS : !C.split;
    C.whole = C.split && !ragged && max_keys <= AT_WHOLE_KEYS;
    C.grid = at_grid(dim, sms);
    if (C.split && !C.whole) C.bytes = (at_desc_bytes(C.grid) + 2 * C.grid * at_part_floats(dim) * 4 + 127) / 128 * 128;
    C.tc_offset = C.bytes;
    C.slices = 1;
    if (C.tc)
    {
        const int rows = ta_rows(dim), kb = dim <= 128 ? 128 : 64;
        C.tiles = (int) (ragged ? all / rows + min((long) seqs, all / (AT_SPLIT_ROWS + 1)) : seqs * ((each + rows - 1) / rows));
        const long keys = window ? min(max_keys, (long) window + sinks + rows / group + 1) : max_keys;
        C.slices = ta_slices((long) C.tiles * kv_heads, (keys + kb - 1) / kb, sms);
        if (C.slices > 1) C.bytes += (size_t) C.tiles * kv_heads * C.slices * ta_part_floats(dim) * 4;
    }
    return C;
}

template <typename T, int D>
static int at_launch(AtPlan& S, cudaStream_t stream)
{
    const amp_attention_args& P = S.P;
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return cuda_rc(e, "attention device");
    if (cudaError_t e = ensure_smem(attention_split_kernel<T, D>, at_smem<D>, dev)) return cuda_rc(e, "attention shared memory");
    const int group = P.heads / P.kv_heads;
    int grid = S.grid;
    if (S.whole) grid = P.seqs * P.kv_heads * ((P.tokens / P.seqs * group + AT_ROWS - 1) / AT_ROWS);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(128, 1, 1);
    cfg.dynamicSmemBytes = at_smem<D>;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = S.pdl ? 1 : 0;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, attention_split_kernel<T, D>, (const AtPlan) S)) return cuda_rc(e, "attention launch");
    if (S.whole || grid < 2) return 0;
    cfg.gridDim = dim3(grid - 1, P.cu ? AT_ROWS : min(AT_ROWS, P.tokens / P.seqs * group), 1);
    cfg.dynamicSmemBytes = 0;
    return cuda_rc(cudaLaunchKernelEx(&cfg, attention_join_kernel<T, D>, (const AtPlan) S), "attention join launch");
}

}  // namespace amp

using namespace amp;

AMP_API long amp_b200_attention_workspace(int tokens, int seqs, int heads, int kv_heads, int dim, int ragged, long max_keys, int window, int sinks)
{
    if (tokens <= 0 || seqs <= 0 || kv_heads <= 0 || heads < kv_heads || (dim != 64 && dim != 128 && dim != 256) || window < 0 || sinks < 0) return 0;
    int rc = 0;
    const AtDevice* d = at_device(&rc);
    if (!d) return rc < 0 ? rc : -1;
    return (long) at_cut(tokens, seqs, heads, kv_heads, dim, ragged != 0, max_keys, min(window, AT_MAX_POS), min(sinks, AT_MAX_POS), d->sms).bytes;
}

AMP_API int amp_b200_attention(const amp_attention_args* args, cudaStream_t stream)
{
    AMP_REQUIRE(args, "attention: null arguments");
    AtPlan S;
    amp_attention_args& P = S.P;
    P = *args;
    if (P.tokens == 0 || P.seqs == 0) return 0;
    AMP_REQUIRE(P.q && P.k_cache && P.v_cache && P.out && (P.table || P.max_pages == 0) && P.pos, "attention: null pointer");
    AMP_REQUIRE(P.tokens > 0 && P.seqs > 0 && P.tokens <= (1 << 24) && P.seqs <= (1 << 20), "attention: %d tokens of %d sequences", P.tokens, P.seqs);
    AMP_REQUIRE(P.cu || P.tokens % P.seqs == 0, "attention: %d tokens do not divide into %d sequences", P.tokens, P.seqs);
    AMP_REQUIRE(P.kv_heads > 0 && P.heads > 0 && P.heads % P.kv_heads == 0 && P.heads <= 1024, "attention: %d heads on %d key-value heads", P.heads, P.kv_heads);
    if (P.dim != 64 && P.dim != 128 && P.dim != 256) return fail(AMP_E_UNSUPPORTED, "attention: head width %d (64, 128 or 256)", P.dim);
    AMP_REQUIRE(P.pages > 0 && P.page_size > 0 && P.max_pages >= 0 && (long long) P.max_pages * P.page_size <= AT_MAX_POS,
                "attention: page sizes (up to 2^30 positions per sequence)");
    AMP_REQUIRE(P.window >= 0 && P.sinks >= 0, "attention: window and sinks must not be negative");
    AMP_REQUIRE(((((uintptr_t) P.q | (uintptr_t) P.k_cache | (uintptr_t) P.v_cache | (uintptr_t) P.out) & 15) |
                 ((P.q_token | P.q_head | P.out_token | P.out_head | P.k_page | P.k_row | P.k_head | P.v_page | P.v_row | P.v_head) & 7)) == 0,
                "attention: pointers must be 16-byte aligned and strides multiples of 8 values");
    AMP_REQUIRE(P.scale == P.scale, "attention: scale is not a number");
    P.window = min(P.window, AT_MAX_POS);
    P.sinks = min(P.sinks, AT_MAX_POS);
    int rc = 0;
    const AtDevice* d = at_device(&rc);
    if (!d) return rc;
    const AtCut C = at_cut(P.tokens, P.seqs, P.heads, P.kv_heads, P.dim, P.cu != nullptr, (long) P.max_pages * P.page_size, P.window, P.sinks, d->sms);
    if (C.bytes)
        AMP_REQUIRE(P.workspace && ((uintptr_t) P.workspace & 15) == 0 && P.workspace_bytes >= (long) C.bytes, "attention: workspace too small or misaligned");
    if (C.split)
    {
        S.grid = C.grid; S.whole = C.whole; S.pdl = g_pdl; S.split_rows = P.cu ? AT_SPLIT_ROWS : 1 << 30;
        S.scale2 = P.scale * 1.4426950408889634f;
        if (P.bf16)
            rc = P.dim == 64 ? at_launch<__nv_bfloat16, 64>(S, stream) : P.dim == 128 ? at_launch<__nv_bfloat16, 128>(S, stream) : at_launch<__nv_bfloat16, 256>(S, stream);
        else
            rc = P.dim == 64 ? at_launch<__half, 64>(S, stream) : P.dim == 128 ? at_launch<__half, 128>(S, stream) : at_launch<__half, 256>(S, stream);
        if (rc) return rc;
    }
    if (!C.tc) return 0;
    TaPlan A;
    A.P = P; A.tiles = C.tiles; A.slices = C.slices; A.split_rows = P.cu ? AT_SPLIT_ROWS : 0; A.pdl = g_pdl;
    A.scale2 = P.scale * 1.4426950408889634f; A.part_offset = C.tc_offset;
    return attention_tc(A, stream);
}
