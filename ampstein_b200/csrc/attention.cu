// Attention of a few new tokens per sequence over a paged key-value cache: one pass over the keys and values, split over the
// cache's length and joined.
//
// The query heads that share a key-value head, times the sequence's new tokens, are the rows of one problem (row = token * group +
// head). A row tile is 16 * WR rows, 16 being the M of mma.sync m16n8k16. The keys that a sequence's new tokens see, counted through
// (the first tokens and the window's, without what lies between), are cut into units. All units of the call, ordered (sequence, head,
// row tile, unit), are cut into equal contiguous ranges, one per CTA: the lengths stand on the device, so that a captured graph replays
// with other lengths, and long and short sequences share the device evenly. What a CTA holds of a (sequence, head, row tile) that other
// CTAs share, a part (o, m, l), goes to the workspace, and a second kernel joins the parts in ascending key order: the same sums in every
// run.
//
// The warps of a CTA are WK groups of WR: a group owns KW keys of every unit, its warps 16 rows each. A group has a ring of half
// stages (KW keys, then their values), filled by its own lanes with 16-byte asynchronous copies, and meets nobody else until the segment
// ends: every warp keeps m, l and o of its rows over its keys. The rings run ahead over the ends of segments.
//
// What bounds it: memory, and a fixed 8 us (launch, positions, table, first keys: 4; the second kernel 4), of which sequences
// that see few keys are spared the second (AT_CLUSTER_KEYS). 32 query heads on 8 key-value heads of 128 values, fp16, us a call in a
// captured chain: one sequence of 128 keys 4.2, 512 5.6, 4000 10.1, 131072 88.6 (6.1 TB/s, 0.94 of the measured copy rate), 32 sequences of
// 2000 keys 51.7 (5.1 TB/s), of 100 to 8192 keys 54.3 (counting the end of a segment as a unit took 71 to 53: a range of
// many short sequences took as long again as its keys). mma.sync and not tcgen05: at 16 rows and 128 values a warp needs 400 issue cycles
// for the 16 KB that a scheduler's share of the memory brings in 2850. 32 keys per step where the registers allow it: the
// look-ups, the row maxima and the loop are per step (32 x 2048 keys, 16 / 32 keys: 60.0 / 53.3). Wide heads keep q in shared
// memory (256 values: 49.7 -> 41.0 for seven sequences of 1000 to 30000 keys).
#include "attention_tc.cuh"

namespace amp {

constexpr int AT_WARP_SEQS = 32;               // sequences that a warp counts by itself

constexpr int AT_WARPS = 4, AT_THREADS = 32 * AT_WARPS;
template <int D> constexpr int at_kw = D == 256 ? 16 : 32;     // keys of a group's step
template <int D> constexpr int at_ctas = D == 64 ? 3 : 2;      // per SM
template <int D> constexpr int at_half_bytes = at_kw<D> * D * 2;
template <int WR> constexpr int at_wk = AT_WARPS / WR;
template <int WR> constexpr int at_rows = 16 * WR;             // of a row tile
template <int D, int WR> constexpr int at_unit = at_wk<WR> * at_kw<D>;         // keys
// shared memory: rings, then the rows of q
template <int D, int WR> constexpr int at_halves = (D == 64 ? 64 : D == 128 ? (WR == 4 ? 80 : 96) : (WR == 1 ? 96 : WR == 2 ? 80 : 64)) * 1024 / (at_wk<WR> * at_half_bytes<D>);
template <int D, int WR> constexpr int at_ring_bytes = at_halves<D, WR> * at_wk<WR> * at_half_bytes<D>;
template <int D, int WR> constexpr int at_smem = at_ring_bytes<D, WR> + at_rows<WR> * D * 2;

struct AtPlan
{
    amp_attention_args P;
    int grid;                                  // CTAs of the split form
    int unit, rows;                            // keys of a unit, rows of a row tile: powers of two
    int unit_shift, rows_shift, cluster_shift;
    int group, group_mul, each;                // heads / kv_heads, ceil(2^16 / group); tokens of every sequence without cu
    int split_rows;                            // with cu: sequences of more rows (tokens x group) are the prompt form's
    int cluster;                               // > 0: every (sequence, head, row tile) belongs to a cluster of so many CTAs, which join in shared memory
    int by_segment;                            // join: blockIdx.x is a segment, else the CTA whose range begins inside it
    int pdl;
    float scale2;                              // scale * log2(e)
    AtPages g;
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

constexpr int AT_MAX_CLUSTER = 8;              // portable

__device__ __forceinline__ void at_cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");      // (a warp's lanes may leave the loop in front one by one)
}

// The same place of shared memory in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t at_map(uint32_t addr, int rank)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ float2 at_ld_cluster2(uint32_t addr)
{
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ float4 at_ld_cluster4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// Row tiles of a sequence, and units of each of them (one at least: a segment without keys stores its zeros). (No division where a shift
// or a product will do: what stands in front of the first load and behind the last is a chain of such steps. us with divisions / so: one
// sequence of 128, 512, 4000 keys 4.9 / 4.3, 6.8 / 5.6, 10.6 / 9.9; 48 windows of 1024 12.7 / 11.3; seven of 1000 to 30000 keys and three tokens,
// 256 values 64 / 56)
__device__ __forceinline__ int at_row_tiles(const AtPlan& S, const AtSeq& s)
{
    const int rows = s.count * S.group;
    return rows > S.split_rows ? 0 : (rows + S.rows - 1) >> S.rows_shift;
}

__device__ __forceinline__ int at_units(const AtPlan& S, const AtKeys& k) { return max(1, (k.count() + S.unit - 1) >> S.unit_shift); }

// Token of a row: row / group, exact for the up to 64 rows of this form (the product is too large by less than row group / 2^16 / group)
__device__ __forceinline__ int at_tok(const AtPlan& S, int row) { return row * S.group_mul >> 16; }

// A place in the order of units. The end of a segment, where its parts meet and the next rows are fetched, counts as one more unit
// (u == units): it takes a CTA about as long, and the many ends of short sequences would come on top of a full range.
struct AtCursor
{
    int b, h, rt, u, tiles, units;
    AtSeq s;
    AtKeys k;

    __device__ __forceinline__ void load(const AtPlan& S)
    {
        s = at_seq(S.P, b, S.each);
        k = at_keys(S.P, s.first, s.count);
        tiles = at_row_tiles(S, s);
        units = at_units(S, k);
    }
    // the at-th unit of sequence b
    __device__ __forceinline__ void place(const AtPlan& S, int seq, int at)
    {
        b = seq;
        load(S);
        const int row_tile = at / (units + 1);
        u = at - row_tile * (units + 1);
        h = tiles == 1 ? row_tile : row_tile / tiles;
        rt = row_tile - h * tiles;
    }
    // to the next unit with keys, or segment; the caller knows that there is one
    __device__ __forceinline__ void advance(const AtPlan& S)
    {
        if (++u < units) return;
        u = 0;
        if (++rt < tiles) return;
        rt = 0;
        if (++h < S.P.kv_heads) return;
        h = 0;
        do { ++b; load(S); } while (!tiles && b + 1 < S.P.seqs);
    }
};

// Units of the sequences, counted (there are fewer than 2^31, the host sees to it). Up to 32 sequences every warp does it by itself,
// one per lane; beyond, the block, a run per thread. All threads of the block call these.
struct AtCount
{
    int b0, b1;                                // this lane's, or thread's, sequences
    int before, mine, total;                   // units in front of them, of them, of all
    bool warp;                                 // counted by the warp
    int ctas, each, more;                      // CTAs with units: the first `more` have each + 1, the others each

    static __device__ __forceinline__ int units_of(const AtPlan& S, int b)
    {
        const AtSeq s = at_seq(S.P, b, S.each);
        return S.P.kv_heads * at_row_tiles(S, s) * (at_units(S, at_keys(S.P, s.first, s.count)) + 1);
    }

    template <int NT>
    __device__ __forceinline__ void count(const AtPlan& S, int* s_scan)
    {
        const int t = threadIdx.x, lane = t & 31;
        warp = S.P.seqs <= AT_WARP_SEQS;
        const int run = warp ? 1 : (S.P.seqs + NT - 1) / NT;
        b0 = min(S.P.seqs, (warp ? lane : t) * run);
        b1 = min(S.P.seqs, b0 + run);
        mine = 0;
        for (int b = b0; b < b1; ++b) mine += units_of(S, b);
        int sum = mine;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        before = sum - mine;
        if (warp) total = __shfl_sync(0xffffffffu, sum, 31);
        else
        {
            if (lane == 31) s_scan[t >> 5] = sum;
            __syncthreads();
            total = 0;
            for (int w = 0; w < NT / 32; ++w) { if (w == t >> 5) before += total; total += s_scan[w]; }
        }
        ctas = min(S.grid, total);
        each = ctas ? total / ctas : 0;
        more = total - each * ctas;
    }

    __device__ __forceinline__ int begin(int cta) const { return cta * each + min(cta, more); }

    // the CTA that has unit u
    __device__ __forceinline__ int cta_of(int u) const
    {
        const int low = more * (each + 1);
        return u < low ? u / (each + 1) : more + (u - low) / each;
    }

    // sequence of unit u (u < total), and the units in front of the sequence
    __device__ __forceinline__ void find(const AtPlan& S, int u, int& b, int& front, int* s_found) const
    {
        const bool here = u >= before && u < before + mine;
        if (warp)
        {
            b = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
            front = __shfl_sync(0xffffffffu, before, b);
            return;
        }
        if (here)
        {
            int at = before;
            for (int i = b0; i < b1; ++i)
            {
                const int n = units_of(S, i);
                if (u < at + n) { s_found[0] = i; s_found[1] = at; break; }
                at += n;
            }
        }
        __syncthreads();
        b = s_found[0];
        front = s_found[1];
    }

    // units in front of sequence b
    __device__ __forceinline__ int front_of(const AtPlan& S, int b, int* s_found) const
    {
        if (warp) return __shfl_sync(0xffffffffu, before, b);
        if (b >= b0 && b < b1)
        {
            int at = before;
            for (int i = b0; i < b; ++i) at += units_of(S, i);
            s_found[0] = at;
        }
        __syncthreads();
        return s_found[0];
    }
};

// Workspace: two parts per CTA (o of the row tile, then m and l of its rows): of the segment that began before the CTA, and of the
// one that it does not end
__host__ __device__ constexpr size_t at_part_floats(int rows, int dim) { return (size_t) rows * (dim + 2); }

template <typename T, int D, int WR, bool CLUSTER>
__global__ __launch_bounds__(AT_THREADS, at_ctas<D>)
void attention_split_kernel(const AtPlan S)
{
    const amp_attention_args& P = S.P;
    constexpr int NT = AT_THREADS, WK = at_wk<WR>, KW = at_kw<D>, H = at_halves<D, WR>, HALF = at_half_bytes<D>;
    constexpr int CH = D / 8, NK = KW / 8, ROWS = at_rows<WR>, UNIT = at_unit<D, WR>;
    constexpr bool KEEP_Q = D <= 128;          // q's fragments stay in registers (256: they are read for every step)
    static_assert(H >= 3, "ring");
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float s_ml[WK][ROWS][2];
    __shared__ int s_scan[AT_WARPS], s_found[2];

    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, grp = warp / WR, wr = warp % WR, cta = blockIdx.x;
    const int group = S.group;
    if (S.pdl) { pdl_wait(); pdl_launch_dependents(); }

    // the CTA's range of units
    AtCursor in;
    int left;
    if (CLUSTER)
    {
        in.b = cta >> S.cluster_shift;
        in.load(S);
        in.h = in.tiles == 1 ? blockIdx.y : blockIdx.y / in.tiles;
        in.rt = blockIdx.y - in.h * in.tiles;
        // (a share may be empty: it then is of a cluster that has more CTAs than units)
        const int rank = cta - (in.b << S.cluster_shift);
        in.u = in.units * rank >> S.cluster_shift;
        left = (in.units * (rank + 1) >> S.cluster_shift) - in.u;
        in.units = in.u + left;                              // the share ends like a segment
        left += left > 0;
    }
    else
    {
        AtCount C;
        C.count<NT>(S, s_scan);
        if (cta >= C.ctas) return;
        const int u0 = C.begin(cta);
        left = C.begin(cta + 1) - u0;
        int b, front;
        C.find(S, u0, b, front, s_found);
        in.place(S, b, u0 - front);
        if (in.u == in.units)                                // (the CTA in front ends that segment)
        {
            if (--left == 0) return;
            in.advance(S);
        }
    }
    const bool began_before = in.u > 0;

    const uint32_t ring = smem_u32(smem) + grp * H * HALF, q_s = smem_u32(smem) + at_ring_bytes<D, WR>;
    auto sync_group = [&]() { if constexpr (WR == 1) __syncwarp(); else asm volatile("bar.sync %0, %1;" :: "r"(1 + grp), "n"(32 * WR) : "memory"); };

    // ---- loads: lane l looks up key l of the group's KW, the table entry a unit ahead; halves alternate keys, values -----------
    AtCursor ld = in;
    int to_load = left;                                      // units
    bool values = false, pre_live = false;
    int pre_page = 0, pre_row = 0, fill_slot = 0;
    const unsigned char* const k_lane = reinterpret_cast<const unsigned char*>(P.k_cache) + lane % CH * 16;
    const unsigned char* const v_lane = reinterpret_cast<const unsigned char*>(P.v_cache) + lane % CH * 16;
    auto look_up = [&]() {
        const int i = ld.u * UNIT + grp * KW + (lane % KW);
        pre_live = i < ld.k.count();
        if (pre_live)
        {
            const int j = ld.k.key(i), pg = S.g.page_of(j);
            pre_row = j - pg * P.page_size;
            pre_page = P.table[(long long) ld.b * P.table_row + pg];
        }
    };
    auto issue = [&]() {
        if (to_load > 0)
        {
            const bool found = (unsigned) pre_page < (unsigned) P.pages;
            const uint32_t off = values ? pre_page * S.g.v_page + pre_row * S.g.v_row : pre_page * S.g.k_page + pre_row * S.g.k_row;
            const unsigned char* const from = values ? v_lane + ld.h * P.v_head * 2 : k_lane + ld.h * P.k_head * 2;
            const uint32_t have = __ballot_sync(0xffffffffu, pre_live && found), at = ring + fill_slot * HALF;
            constexpr int PER = CH >= 32 ? 1 : 32 / CH;      // rows per warp-wide copy
            const int r_lane = wr * (KW / WR) + (CH >= 32 ? 0 : lane / CH);
            if (have == 0xffffffffu)
            {
                #pragma unroll
                for (int r0 = 0; r0 < KW / WR; r0 += PER)
                {
                    const int r = r_lane + r0;
                    cp_async16_s(at + r * (2 * D) + (((lane % CH) ^ (r & 7)) << 4), from + (unsigned long long) __shfl_sync(0xffffffffu, off, r) * 16);
                }
            }
            else
            {
                // behind the last key, and on pages outside the pool: zeros
                #pragma unroll
                for (int r0 = 0; r0 < KW / WR; r0 += PER)
                {
                    const int r = r_lane + r0;
                    const uint32_t o = __shfl_sync(0xffffffffu, off, r);
                    const bool get = (have >> r) & 1;
                    at_copy16(at + r * (2 * D) + (((lane % CH) ^ (r & 7)) << 4), get ? from + (unsigned long long) o * 16 : from, get);
                }
                const uint32_t lost = __ballot_sync(0xffffffffu, pre_live && !found);
                if (lost && !values)
                {
                    // a key that cannot be found is NaN to the rows that see it, its value 0 (the copies of zeros are in front)
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    __syncwarp();
                    for (int i = lane; i < KW / WR * CH; i += 32)
                    {
                        const int r = wr * (KW / WR) + i / CH;
                        if ((lost >> r) & 1)
                            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" :: "r"(at + r * (2 * D) + (i % CH) * 16), "r"(0x7fff7fffu) : "memory");
                    }
                }
            }
            if (values)
            {
                to_load -= ld.u + 1 == ld.units ? 2 : 1;
                if (to_load > 0) { ld.advance(S); look_up(); }
            }
            values = !values;
        }
        cp_async_commit();
        fill_slot = fill_slot + 1 == H ? 0 : fill_slot + 1;
    };
    look_up();

    // ---- the segments of the range, a half stage per turn ---------------------------------------------------------------------
    uint32_t qf[KEEP_Q ? D / 16 : 1][4], pf[NK / 2][4];
    float o[D / 8][4], m[2], l[2];
    int n0[2], c1[2], len[2];                                // keys that the lane's two rows see: [0, n0) and [c1, c1 + len]
    int whole_from = 0, whole_to = 0;                        // keys that all rows see
    bool fresh = true, first_segment = true, hold = false;
    int slot = 0, key_slot = 0, ahead = 0;                   // ahead: half stages requested from the one at hand on
    // fragment of q for a step of 16 values: rows of the warp
    auto q_fragment = [&](int ks, uint32_t (&f)[4]) {
        const int r = wr * 16 + (lane & 15), c = 2 * ks + (lane >> 4);
        at_ldsm4(q_s + r * (2 * D) + ((c ^ (r & 7)) << 4), f);
    };
    for (int turn = -1; left > 0; ++turn)
    {
        // the half at hand has landed, for all lanes of the group; the ones in front of it are read: their slots are filled again
        if (turn >= 0)
        {
            if (ahead == H) asm volatile("cp.async.wait_group %0;" :: "n"(H - 1) : "memory");
            else if (ahead == H - 1) asm volatile("cp.async.wait_group %0;" :: "n"(H - 2) : "memory");
            else asm volatile("cp.async.wait_group %0;" :: "n"(H - 3) : "memory");
            sync_group();
        }
        const bool is_key = (turn & 1) == 0, ends = in.u + 1 == in.units;
        hold = !is_key && turn >= 0 && (ends || left == 1);  // (the end of a segment uses both halves at hand)
        #pragma unroll 1
        while (ahead < H && !hold) { issue(); ++ahead; }
        if (turn < 0) continue;
        const int key0 = in.u * UNIT + grp * KW;
        const bool some = key0 < in.k.count();
        const uint32_t at = ring + slot * HALF;
        if (is_key)
        {
            if (fresh)
            {
                for (int i = t; i < ROWS * CH; i += NT)
                {
                    const int r = i / CH, c = i % CH, row = in.rt * ROWS + r, tok = at_tok(S, row);
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (tok < in.s.count)
                        v = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(P.q) + (long long) (in.s.row0 + tok) * P.q_token
                                                            + (long long) (in.h * group + row - tok * group) * P.q_head + c * 8);
                    *reinterpret_cast<uint4*>(smem + at_ring_bytes<D, WR> + r * (2 * D) + ((c ^ (r & 7)) << 4)) = v;
                }
                #pragma unroll
                for (int i = 0; i < 2; ++i)
                {
                    m[i] = -INFINITY;
                    l[i] = 0.0f;
                    at_row_keys(P, in.k, in.s.first + at_tok(S, in.rt * ROWS + wr * 16 + (lane >> 2) + 8 * i), n0[i], c1[i], len[i]);
                }
                at_whole_keys(P, in.k, in.s.first, in.s.first + in.s.count - 1, whole_from, whole_to);
                #pragma unroll
                for (int n = 0; n < D / 8; ++n) { o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f; }
                __syncthreads();
                if constexpr (KEEP_Q)
                {
                    #pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) q_fragment(ks, qf[ks]);
                }
                fresh = false;
            }
            key_slot = slot;
            if (some)
            {
                // s = q k^T: rows x KW keys
                float s[NK][4];
                #pragma unroll
                for (int n = 0; n < NK; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
                #pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                {
                    if constexpr (!KEEP_Q) q_fragment(ks, qf[0]);
                    #pragma unroll
                    for (int n = 0; n < NK; n += 2)
                    {
                        const int r = n * 8 + (lane & 7) + ((lane >> 4) << 3), c = 2 * ks + ((lane >> 3) & 1);
                        uint32_t f[4];
                        at_ldsm4(at + r * (2 * D) + ((c ^ (r & 7)) << 4), f);
                        at_mma<T>(s[n], qf[KEEP_Q ? ks : 0], f[0], f[1]);
                        at_mma<T>(s[n + 1], qf[KEEP_Q ? ks : 0], f[2], f[3]);
                    }
                }
                const bool all = key0 >= whole_from && key0 + KW <= whole_to;
                float top[2] = { m[0], m[1] };
                #pragma unroll
                for (int n = 0; n < NK; ++n)
                {
                    #pragma unroll
                    for (int e = 0; e < 4; ++e)
                    {
                        s[n][e] *= S.scale2;
                        if (!all)
                        {
                            const int c = key0 + n * 8 + (lane & 3) * 2 + (e & 1), i = e >> 1;
                            if (!(c < n0[i] || (uint32_t) (c - c1[i]) <= (uint32_t) len[i])) s[n][e] = -INFINITY;
                        }
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
                        const float f = top[i] > m[i] ? (m[i] == -INFINITY ? 0.0f : at_exp2(at_base<T>(m[i]) - at_base<T>(top[i]))) : 1.0f;
                        m[i] = top[i];
                        l[i] *= f;
                        #pragma unroll
                        for (int n = 0; n < D / 8; ++n) { o[n][2 * i] *= f; o[n][2 * i + 1] *= f; }
                    }
                }
                const float base0 = m[0] == -INFINITY ? 0.0f : at_base<T>(m[0]), base1 = m[1] == -INFINITY ? 0.0f : at_base<T>(m[1]);
                float sum[2] = { 0.0f, 0.0f };               // (by itself: small weights beside a large l are lost one by one)
                #pragma unroll
                for (int n = 0; n < NK; ++n)
                {
                    s[n][0] = at_exp2(s[n][0] - base0); s[n][1] = at_exp2(s[n][1] - base0);
                    s[n][2] = at_exp2(s[n][2] - base1); s[n][3] = at_exp2(s[n][3] - base1);
                    sum[0] += s[n][0] + s[n][1];
                    sum[1] += s[n][2] + s[n][3];
                    pf[n / 2][2 * (n & 1)] = AtType<T>::pack(s[n][0], s[n][1]);
                    pf[n / 2][2 * (n & 1) + 1] = AtType<T>::pack(s[n][2], s[n][3]);
                }
                l[0] += sum[0];
                l[1] += sum[1];
            }
        }
        else
        {
            // values without a finite magnitude, of keys that not all rows see (12.4 -> 12.8 us for eight sequences of three tokens in windows of 512)
            if (some && in.s.count > 1 && (key0 < whole_from || min(key0 + KW, in.k.count()) > whole_to))
            {
                uint32_t odd = 0;
                #pragma unroll 4
                for (int i = lane; i < KW * CH; i += 32) odd |= at_odd<T>(at_lds16(at + i * 16));
                if (__any_sync(0xffffffffu, odd))
                {
                    #pragma unroll 1
                    for (int r = 0; r < KW; ++r)
                    {
                        const int c = key0 + r;
                        const bool see0 = c < n0[0] || (uint32_t) (c - c1[0]) <= (uint32_t) len[0], see1 = c < n0[1] || (uint32_t) (c - c1[1]) <= (uint32_t) len[1];
                        #pragma unroll
                        for (int n = 0; n < D / 8; ++n)
                        {
                            uint32_t x;
                            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at + r * (2 * D) + ((n ^ (r & 7)) << 4) + (lane & 3) * 4) : "memory");
                            const uint32_t is = AtType<T>::odd(x);
                            const float2 v = AtType<T>::unpack(x);
                            if (is & 0x8000u) { o[n][0] += see0 ? v.x : 0.0f; o[n][2] += see1 ? v.x : 0.0f; }
                            if (is & 0x80000000u) { o[n][1] += see0 ? v.y : 0.0f; o[n][3] += see1 ? v.y : 0.0f; }
                        }
                    }
                    sync_group();                            // (all warps of the group have looked)
                    for (int i = lane + 32 * wr; i < KW * CH; i += 32 * WR) at_sts16_even<T>(at + i * 16, at_lds16(at + i * 16));
                    sync_group();
                }
            }
            if (some)
            {
                #pragma unroll
                for (int kk = 0; kk < NK / 2; ++kk)
                {
                    #pragma unroll
                    for (int n = 0; n < D / 16; ++n)
                    {
                        const int r = kk * 16 + (lane & 15), c = 2 * n + (lane >> 4);
                        uint32_t f[4];
                        at_ldsm4_trans(at + r * (2 * D) + ((c ^ (r & 7)) << 4), f);
                        at_mma<T>(o[2 * n], pf[kk], f[0], f[1]);
                        at_mma<T>(o[2 * n + 1], pf[kk], f[2], f[3]);
                    }
                }
            }
            left -= ends ? 2 : 1;
            if (hold)
            {
                const bool before = first_segment && began_before, shared = CLUSTER ? S.cluster > 1 : before || !ends;
                // (a cluster's part stays in shared memory, behind the rows of q)
                float* const part = CLUSTER ? reinterpret_cast<float*>(smem + at_smem<D, WR>)
                                            : reinterpret_cast<float*>(P.workspace) + (size_t) (2 * cta + (before ? 0 : 1)) * at_part_floats(ROWS, D);
                #pragma unroll
                for (int i = 0; i < 2; ++i)
                {
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
                    m[i] = at_base<T>(m[i]);                 // (what the sums count from)
                    if ((lane & 3) == 0) { s_ml[grp][wr * 16 + (lane >> 2) + 8 * i][0] = m[i]; s_ml[grp][wr * 16 + (lane >> 2) + 8 * i][1] = l[i]; }
                }
                __syncthreads();
                float f[2];
                #pragma unroll
                for (int i = 0; i < 2; ++i)
                {
                    float top = s_ml[0][wr * 16 + (lane >> 2) + 8 * i][0];
                    #pragma unroll
                    for (int g = 1; g < WK; ++g) top = fmaxf(top, s_ml[g][wr * 16 + (lane >> 2) + 8 * i][0]);
                    f[i] = m[i] == -INFINITY ? 0.0f : at_exp2(m[i] - top);
                }
                // the groups' parts meet in the two half stages that each has just read, D / WR columns at a time: the columns of a row
                // are turned round by 8 for every row (mod 4), so that eight rows meet all banks
                constexpr int COLS = D / WR, PIECE = 16 * COLS * 4, TURN = COLS >= 32 ? 3 : COLS / 8 - 1;
                auto place = [&](int g, int w, int r, int c) {           // byte offset in the group's ring
                    const int x = w * PIECE + (r * COLS + (c ^ ((r & TURN) << 3))) * 4;
                    return g * H * HALF + (x < HALF ? key_slot * HALF + x : slot * HALF + x - HALF);
                };
                #pragma unroll
                for (int pass = 0; pass < WR; ++pass)
                {
                    #pragma unroll
                    for (int i = 0; i < 2; ++i)
                    {
                        const int r = (lane >> 2) + 8 * i;
                        #pragma unroll
                        for (int n = 0; n < COLS / 8; ++n)
                            *reinterpret_cast<float2*>(smem + place(grp, wr, r, n * 8 + (lane & 3) * 2)) =
                                make_float2(o[pass * (COLS / 8) + n][2 * i] * f[i], o[pass * (COLS / 8) + n][2 * i + 1] * f[i]);
                    }
                    __syncthreads();
                    #pragma unroll 1
                    for (int i = t; i < ROWS * COLS / 4; i += NT)
                    {
                        const int r = i / (COLS / 4), c = (i % (COLS / 4)) * 4;
                        const int row = in.rt * ROWS + r, tok = at_tok(S, row);
                        if (tok >= in.s.count) break;        // (rows ascend with i)
                        float top = s_ml[0][r][0], sum = 0.0f;
                        #pragma unroll
                        for (int g = 1; g < WK; ++g) top = fmaxf(top, s_ml[g][r][0]);
                        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        #pragma unroll
                        for (int g = 0; g < WK; ++g)
                        {
                            sum += s_ml[g][r][0] == -INFINITY ? s_ml[g][r][1] : s_ml[g][r][1] * at_exp2(s_ml[g][r][0] - top);      // (an l of NaN stays one)
                            const float4 y = *reinterpret_cast<const float4*>(smem + place(g, r >> 4, r & 15, c));
                            x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
                        }
                        const int col = pass * COLS + c;
                        if (shared)
                        {
                            *reinterpret_cast<float4*>(part + r * D + col) = x;
                            if (col == 0) *reinterpret_cast<float2*>(part + ROWS * D + 2 * r) = make_float2(top, sum);
                        }
                        else
                            at_store<T>(P, in.s, tok, in.h * group + row - tok * group, col, x, top, sum);
                    }
                    __syncthreads();
                }
                fresh = true;
                first_segment = false;
            }
            if (left > 0) in.advance(S);
        }
        slot = slot + 1 == H ? 0 : slot + 1;
        --ahead;
    }

    if (CLUSTER && S.cluster > 1)
    {
        // every CTA of the cluster finishes its share of the segment's values, in order of the keys. (The barrier in front: all parts are
        // there, and all CTAs run. The one behind: nobody leaves with a part that is still read.)
        const int C = S.cluster, units = at_units(S, in.k), per = (ROWS * D / 4) >> S.cluster_shift, rank = cta & (C - 1);
        at_cluster_sync();
        const uint32_t mine = smem_u32(smem) + at_smem<D, WR>;
        for (int i = rank * per + t; i < (rank + 1) * per; i += NT)
        {
            const int r = i / (D / 4), c = (i % (D / 4)) * 4, row = in.rt * ROWS + r, tok = at_tok(S, row);
            if (tok >= in.s.count) break;
            float m = -INFINITY, l = 0.0f;
            float2 ml[AT_MAX_CLUSTER];
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y[AT_MAX_CLUSTER];
            #pragma unroll
            for (int k = 0; k < AT_MAX_CLUSTER; ++k)
            {
                // (an empty share has no part)
                const bool part = k < C && units * k >> S.cluster_shift < units * (k + 1) >> S.cluster_shift;
                ml[k] = part ? at_ld_cluster2(at_map(mine + (ROWS * D + 2 * r) * 4, k)) : make_float2(-INFINITY, 0.0f);
                y[k] = part ? at_ld_cluster4(at_map(mine + (r * D + c) * 4, k)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                m = fmaxf(m, ml[k].x);
            }
            const float base = m == -INFINITY ? 0.0f : m;
            #pragma unroll
            for (int k = 0; k < AT_MAX_CLUSTER; ++k)
            {
                const float f = at_exp2(ml[k].x - base);
                l += ml[k].x == -INFINITY ? ml[k].y : ml[k].y * f;           // (an l of NaN stays one)
                x.x += y[k].x * f; x.y += y[k].y * f; x.z += y[k].z * f; x.w += y[k].w * f;
            }
            at_store<T>(P, in.s, tok, in.h * group + row - tok * group, c, x, m, l);
        }
        at_cluster_sync();
    }
}

// Joins the parts of a segment, row blockIdx.y of it (LOOP: every gridDim.y-th from there): of segment blockIdx.x, or of the one that the range of
// CTA blockIdx.x is the second to hold. (Which parts those are is found behind the wait: in front of it a call took 1.0 to 1.4 us less, but what is
// read for that, positions and lengths, is only visible behind it.)
template <typename T, int D, bool LOOP>
__global__ __launch_bounds__(128)
void attention_join_kernel(const AtPlan S)
{
    const amp_attention_args& P = S.P;
    __shared__ float s_red[4], s_sum[4];
    __shared__ float4 s_o[4][D / 4];
    __shared__ int s_scan[4], s_found[2];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, group = S.group;
    if (S.pdl) { pdl_wait(); pdl_launch_dependents(); }
    AtCount C;
    C.count<128>(S, s_scan);
    AtCursor in;
    int g0;                                                  // first unit of the segment
    int first, last;                                         // CTAs that hold it
    bool join = false;
    if (S.by_segment)
    {
        const int tiles = (S.each * group + S.rows - 1) >> S.rows_shift, at = tiles == 1 ? blockIdx.x : blockIdx.x / tiles, b = at / P.kv_heads;
        in.b = b; in.h = at - b * P.kv_heads; in.rt = blockIdx.x - at * tiles;
        in.load(S);
        g0 = C.front_of(S, b, s_found) + (in.h * in.tiles + in.rt) * (in.units + 1);
        join = true;
    }
    else if ((int) blockIdx.x < C.ctas)
    {
        const int u0 = C.begin(blockIdx.x);
        int b, front;
        C.find(S, u0, b, front, s_found);
        in.place(S, b, u0 - front);
        g0 = u0 - in.u;
        join = in.u > 0 && in.u < in.units;
    }
    if (join)
    {
        first = C.cta_of(g0);
        last = C.cta_of(g0 + in.units - 1);
        join = first < last && (S.by_segment || first == (int) blockIdx.x - 1);
    }
    if (!join) return;

    // part i of the segment: the first is the end of its CTA's range, the others are the beginning of theirs
    const size_t size = at_part_floats(S.rows, D);
    const float* const parts = reinterpret_cast<const float*>(P.workspace);
    const int n = last - first + 1;
    auto part = [&](int i) { return parts + (size_t) (2 * (first + i) + (i ? 0 : 1)) * size; };
    for (int r = blockIdx.y; r < (LOOP ? S.rows : (int) blockIdx.y + 1); r += gridDim.y)
    {
        const int row = in.rt * S.rows + r, tok = at_tok(S, row);
        if (tok >= in.s.count) return;
        float m = -INFINITY;
        for (int i = t; i < n; i += 128) m = fmaxf(m, part(i)[(size_t) S.rows * D + 2 * r]);
        // a warp adds every fourth part up, a lane D / 32 values of the row (in pieces of four); the first parts are on their way while m is found
        constexpr int PIECES = D / 4, EACH = (PIECES + 31) / 32, AHEAD = D == 256 ? 4 : 8;
        float4 x[AHEAD][EACH];
        float2 ml[AHEAD];
        auto fetch = [&](int i0) {
            #pragma unroll
            for (int a = 0; a < AHEAD; ++a)
            {
                const int i = i0 + 4 * a;
                ml[a] = make_float2(-INFINITY, 0.0f);
                if (i >= n) continue;
                const float* p = part(i);
                ml[a] = *reinterpret_cast<const float2*>(p + (size_t) S.rows * D + 2 * r);
                #pragma unroll
                for (int e = 0; e < EACH; ++e)
                    if (PIECES % 32 == 0 || lane + 32 * e < PIECES) x[a][e] = reinterpret_cast<const float4*>(p + r * D)[lane + 32 * e];
            }
        };
        fetch(warp);
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) s_red[warp] = m;
        __syncthreads();
        m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
        const float base = m == -INFINITY ? 0.0f : m;
        float4 acc[EACH];
        #pragma unroll
        for (int e = 0; e < EACH; ++e) acc[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
        for (int i0 = warp; i0 < n; i0 += 4 * AHEAD)
        {
            #pragma unroll
            for (int a = 0; a < AHEAD; ++a)
            {
                if (i0 + 4 * a >= n) continue;
                const float f = at_exp2(ml[a].x - base);
                l += ml[a].x == -INFINITY ? ml[a].y : ml[a].y * f;       // (an l of NaN stays one)
                #pragma unroll
                for (int e = 0; e < EACH; ++e)
                {
                    acc[e].x += x[a][e].x * f; acc[e].y += x[a][e].y * f; acc[e].z += x[a][e].z * f; acc[e].w += x[a][e].w * f;
                }
            }
            if (i0 + 4 * AHEAD < n) fetch(i0 + 4 * AHEAD);
        }
        if (lane == 0) s_sum[warp] = l;
        #pragma unroll
        for (int e = 0; e < EACH; ++e) if (PIECES % 32 == 0 || lane + 32 * e < PIECES) s_o[warp][lane + 32 * e] = acc[e];
        __syncthreads();
        l = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
        for (int c = t; c < PIECES; c += 128)
        {
            float4 y = s_o[0][c];
            #pragma unroll
            for (int w = 1; w < 4; ++w) { const float4 z = s_o[w][c]; y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w; }
            at_store<T>(P, in.s, tok, in.h * group + row - tok * group, c * 4, y, m, l);
        }
        if constexpr (LOOP) __syncthreads();
        else return;
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

// Sequences that see few keys are not cut into ranges: a cluster of up to eight CTAs has each of their segments and joins in shared memory, no
// second kernel follows. Up to AT_WHOLE_KEYS however many segments there are, beyond where at least two CTAs find places for each (the
// lengths may differ). us, equal ranges / this, when both still divided (each is about 1 us faster since; 32 query heads on 8 key-value heads of 128 values): one sequence of 512 and 1024 keys 8.1 / 6.6
// and 8.4 / 7.0, of 2048 8.9 / 9.0; four of 300 and 2000 11.5 / 9.4 and 14.6 / 12.8; 32 of 300 19.1 / 13.0; but 32 of 50 to 2000 keys,
// a CTA each, 29.6 / 39.4. (Equal ranges take 1.2 more again since their second kernel waits before it looks anything up.)
constexpr int AT_WHOLE_KEYS = 512, AT_CLUSTER_KEYS = 2048;
// Rows (tokens x group) up to which a sequence takes the split form, whose ranges follow the lengths; beyond, the prompt form
constexpr int AT_SPLIT_ROWS = 64;

constexpr long AT_SM_BYTES = 228 * 1024;       // of shared memory, per SM

template <int D> static int at_smem_rows(int wr) { return wr == 1 ? at_smem<D, 1> : wr == 2 ? at_smem<D, 2> : at_smem<D, 4>; }
static int at_smem_bytes(int dim, int wr) { return dim == 64 ? at_smem_rows<64>(wr) : dim == 128 ? at_smem_rows<128>(wr) : at_smem_rows<256>(wr); }

static int at_unit_keys(int dim, int wr) { return AT_WARPS / wr * (dim == 64 ? at_kw<64> : dim == 128 ? at_kw<128> : at_kw<256>); }
static int at_grid(int dim, int sms) { return sms * (dim == 64 ? at_ctas<64> : dim == 128 ? at_ctas<128> : at_ctas<256>); }

// How a call is cut up: by its sizes alone (the lengths are on the device)
struct AtCut
{
    bool split, tc;                            // forms that are launched
    int cluster, grid, wr;                     // split form: CTAs per segment (0: equal ranges), CTAs, 16 * wr rows per row tile
    int nq, tiles, slices;                     // prompt form
    size_t tc_offset, bytes;                   // of the workspace
};

// Slices of the keys of each of `items` row tiles, `kt` key tiles long at most: waves of CTAs, each its share of the key tiles and a
// set-up of about two, and a join worth four
static int ta_slices(long items, long kt, int places)
{
    int best = 1;
    double cost = 1e30;
    for (int s = 1; s <= kt && s * items <= 4l * places && s <= 256; ++s)
    {
        const double c = (double) ((items * s + places - 1) / places) * ((double) ((kt + s - 1) / s) + 2) + (s > 1 ? 4 : 0);
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
    C.grid = at_grid(dim, sms);
    const long rows = ragged ? group : each;   // (ragged: single tokens are the rule)
    C.wr = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    const long seen = window ? min(max_keys, (long) window + sinks + tokens / seqs) : max_keys;
    if (C.split && !ragged && seen <= AT_CLUSTER_KEYS)
    {
        const long segments = seqs * kv_heads * ((each + 16 * C.wr - 1) / (16 * C.wr)), unit = at_unit_keys(dim, C.wr);
        const long places = sms * min((long) C.grid / sms, AT_SM_BYTES / (at_smem_bytes(dim, C.wr) + (long) at_part_floats(16 * C.wr, dim) * 4 + 2048));
        for (C.cluster = 1; C.cluster < AT_MAX_CLUSTER && 2 * C.cluster * segments <= places && 2 * C.cluster * unit < seen + unit; C.cluster *= 2) { }
        if (C.cluster == 1 && seen > AT_WHOLE_KEYS) C.cluster = 0;
    }
    if (C.split && !C.cluster) C.bytes = (2 * C.grid * at_part_floats(16 * C.wr, dim) * 4 + 127) / 128 * 128;
    C.tc_offset = C.bytes;
    C.slices = 1;
    if (C.tc)
    {
        // One row tile per CTA and two CTAs per SM where a tile has few keys: set-up and ends of one run under the other's keys. Two row tiles
        // per CTA share every key otherwise (us, one tile / two; 4 query heads per key-value head at 128 values, 8 at 64: windows of 128,
        // 512, 1024, 2048 keys 34.0 / 52.4, 52.6 / 69.6, 76.7 / 91.3, 93.2 / 91.8 at 128; 45.5 / 64.1, 75.1 / 85.3, 113 / 113, 153 / 136 at 64;
        // a prompt of 2048 tokens 53.6 / 56.6 and 88 / 79, of 8192 567 / 509 and 1017 / 747)
        const long few = dim == 128 ? 1536 : 768;
        C.nq = dim == 256 || (window ? min(max_keys, (long) window + sinks + 128 / group) : max_keys) <= few ? 1 : 2;
        const int tile = 128 * C.nq, kb = 64 * C.nq;
        C.tiles = (int) (ragged ? all / tile + min((long) seqs, all / (AT_SPLIT_ROWS + 1)) : seqs * ((each + tile - 1) / tile));
        const long keys = window ? min(max_keys, (long) window + sinks + tile / group + 1) : max_keys;
        C.slices = ta_slices((long) C.tiles * kv_heads, (keys + kb - 1) / kb, C.nq == 1 && dim <= 128 ? 2 * sms : sms);
        if (C.slices > 1) C.bytes += (size_t) C.tiles * kv_heads * C.slices * ta_part_floats(tile, dim) * 4;
    }
    return C;
}

template <typename T, int D, int WR, bool CLUSTER>
static int at_launch(AtPlan& S, cudaStream_t stream)
{
    const amp_attention_args& P = S.P;
    // (a cluster's part)
    const int bytes = at_smem<D, WR> + (CLUSTER && S.cluster > 1 ? (int) at_part_floats(at_rows<WR>, D) * 4 : 0);
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return cuda_rc(e, "attention device");
    if (cudaError_t e = ensure_smem(attention_split_kernel<T, D, WR, CLUSTER>, bytes, dev)) return cuda_rc(e, "attention shared memory");
    S.unit = at_unit<D, WR>;
    S.rows = 16 * WR;
    static_assert((at_unit<D, WR> & (at_unit<D, WR> - 1)) == 0 && (WR & (WR - 1)) == 0, "shifts");
    S.unit_shift = __builtin_ctz(S.unit); S.rows_shift = __builtin_ctz(S.rows); S.cluster_shift = CLUSTER ? __builtin_ctz(S.cluster) : 0;
    const long group = P.heads / P.kv_heads;
    S.group = (int) group; S.group_mul = (int) ((65536 + group - 1) / group); S.each = P.tokens / P.seqs;
    // (segments of the call, where the host knows them)
    const long rows = (long) (P.tokens / P.seqs) * group, segments = (long) P.seqs * P.kv_heads * ((rows + S.rows - 1) / S.rows);
    const long grid = CLUSTER ? (long) P.seqs * S.cluster : S.grid;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    int attrs = S.pdl ? 1 : 0;
    if (CLUSTER && S.cluster > 1)
    {
        attr[attrs].id = cudaLaunchAttributeClusterDimension;
        attr[attrs].val.clusterDim.x = S.cluster;
        attr[attrs].val.clusterDim.y = attr[attrs].val.clusterDim.z = 1;
        ++attrs;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) grid, CLUSTER ? (unsigned) (segments / P.seqs) : 1, 1);
    cfg.blockDim = dim3(AT_THREADS, 1, 1);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = attrs;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, attention_split_kernel<T, D, WR, CLUSTER>, (const AtPlan) S)) return cuda_rc(e, "attention launch");
    if (CLUSTER) return 0;
    cfg.numAttrs = S.pdl ? 1 : 0;
    S.by_segment = !P.cu && segments < S.grid;
    // a row per CTA; with cu there may be up to 64 of them and most CTAs have none: four CTAs go through all (2333 tokens of six prompts,
    // none of which is the split form's: 49.1 us with a row per CTA, 44.4)
    cfg.gridDim = dim3(S.by_segment ? (unsigned) segments : S.grid, P.cu ? 4 : (unsigned) min((long) S.rows, rows), 1);
    cfg.blockDim = dim3(128, 1, 1);
    cfg.dynamicSmemBytes = 0;
    return cuda_rc(P.cu ? cudaLaunchKernelEx(&cfg, attention_join_kernel<T, D, true>, (const AtPlan) S)
                        : cudaLaunchKernelEx(&cfg, attention_join_kernel<T, D, false>, (const AtPlan) S), "attention join launch");
}

template <typename T, int D>
static int at_launch_rows(AtPlan& S, int wr, cudaStream_t stream)
{
    if (S.cluster) return wr == 1 ? at_launch<T, D, 1, true>(S, stream) : wr == 2 ? at_launch<T, D, 2, true>(S, stream) : at_launch<T, D, 4, true>(S, stream);
    return wr == 1 ? at_launch<T, D, 1, false>(S, stream) : wr == 2 ? at_launch<T, D, 2, false>(S, stream) : at_launch<T, D, 4, false>(S, stream);
}

template <typename T>
static int at_launch_dim(AtPlan& S, int wr, cudaStream_t stream)
{
    return S.P.dim == 64 ? at_launch_rows<T, 64>(S, wr, stream) : S.P.dim == 128 ? at_launch_rows<T, 128>(S, wr, stream) : at_launch_rows<T, 256>(S, wr, stream);
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
    AMP_REQUIRE(std::isfinite(P.scale * 1.4426950408889634f), "attention: scale is not finite");
    {
        // (other CTAs may still read what one writes)
        const Span q(P.q, P.dim * 2l, { { P.tokens, P.q_token * 2 }, { P.heads, P.q_head * 2 } }), out(P.out, P.dim * 2l, { { P.tokens, P.out_token * 2 }, { P.heads, P.out_head * 2 } });
        const Span k(P.k_cache, P.dim * 2l, { { P.pages, P.k_page * 2 }, { P.page_size, P.k_row * 2 }, { P.kv_heads, P.k_head * 2 } });
        const Span v(P.v_cache, P.dim * 2l, { { P.pages, P.v_page * 2 }, { P.page_size, P.v_row * 2 }, { P.kv_heads, P.v_head * 2 } });
        AMP_REQUIRE(apart(out, q) && apart(out, k) && apart(out, v), "attention: out overlaps q or a cache");
        const Span lse(P.lse, P.lse ? (long) P.tokens * P.heads * 4 : 0, {});
        AMP_REQUIRE(!P.lse || (apart(lse, out) && apart(lse, q) && apart(lse, k) && apart(lse, v)), "attention: lse overlaps out, q or a cache");
    }
    P.window = min(P.window, AT_MAX_POS);
    P.sinks = min(P.sinks, AT_MAX_POS);
    int rc = 0;
    const AtDevice* d = at_device(&rc);
    if (!d) return rc;
    AtPages g;
    AMP_REQUIRE(at_pages(P, g), "attention: a cache of more than 64 GB, or negative strides");
    const AtCut C = at_cut(P.tokens, P.seqs, P.heads, P.kv_heads, P.dim, P.cu != nullptr, (long) P.max_pages * P.page_size, P.window, P.sinks, d->sms);
    if (C.bytes)
        AMP_REQUIRE(P.workspace && ((uintptr_t) P.workspace & 15) == 0 && P.workspace_bytes >= (long) C.bytes, "attention: workspace too small or misaligned");
    if (C.split)
    {
        // units are counted in 32 bits (whatever cu holds, a sequence has at most AT_SPLIT_ROWS rows there)
        const long group = P.heads / P.kv_heads, rows = 16 * C.wr;
        const double tiles = P.cu ? (double) P.seqs * ((min((long) AT_SPLIT_ROWS, P.tokens * group) + rows - 1) / rows) : (double) (P.tokens * group / rows + P.seqs);
        AMP_REQUIRE(P.kv_heads * tiles * (P.max_pages * (double) P.page_size / at_unit_keys(P.dim, C.wr) + 2) < 2147483648.0,
                    "attention: more keys than one call takes (%d sequences of up to %ld)", P.seqs, (long) P.max_pages * P.page_size);
    }
    if (C.tc)
    {
        // (rows and CTAs are divided in 30 bits)
        AMP_REQUIRE((double) P.tokens * (P.heads / P.kv_heads) + 512 < 1073741824.0 && (double) C.tiles * C.slices * P.kv_heads < 1073741824.0, "attention: too many tokens in one call");
        // (each form waits for the one in front: positions and lengths may come from the launch before the call, and only a grid's own wait makes
        // them visible to it. us in a graph with the few-token form begun under the prompt form's end / so: 64 single tokens of 1000 keys beside
        // a prompt of 2048 tokens 115 / 125, 16 of 4000 beside 64 tokens on 6000 98 / 104; in the other order level)
        TaPlan A;
        A.P = P; A.nq = C.nq; A.tiles = C.tiles; A.slices = C.slices; A.split_rows = P.cu ? AT_SPLIT_ROWS : 0; A.pdl = g_pdl;
        A.scale2 = P.scale * 1.4426950408889634f; A.part_offset = C.tc_offset; A.g = g;
        if ((rc = attention_tc(A, stream))) return rc;
    }
    if (!C.split) return 0;
    S.grid = C.grid; S.cluster = C.cluster; S.pdl = g_pdl; S.split_rows = P.cu ? AT_SPLIT_ROWS : 1 << 30;
    S.scale2 = P.scale * 1.4426950408889634f; S.g = g;
    return P.bf16 ? at_launch_dim<__nv_bfloat16>(S, C.wr, stream) : at_launch_dim<__half>(S, C.wr, stream);
}
