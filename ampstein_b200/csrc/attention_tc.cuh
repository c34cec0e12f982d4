// Launch interface of the prompt form of the attention (attention_tc.cu)
#pragma once
#include "attention.cuh"

namespace amp {

// A CTA has NQ tiles of 128 rows: two, one CTA per SM, or one; then two CTAs share an SM, up to 128 values per head
template <int NQ> constexpr int ta_rows = 128 * NQ;
template <int NQ> constexpr int ta_kb = 64 * NQ;               // keys per tile
template <int NQ> constexpr int ta_threads = 128 * (NQ + 1);
template <int D, int NQ> constexpr int ta_ctas = NQ == 1 && D <= 128 ? 2 : 1;
template <int D, int NQ> constexpr int ta_stages = D == 64 && NQ == 2 ? 8 : 5;         // tiles of keys or values in shared memory
template <int D, int NQ> constexpr int ta_smem = ta_rows<NQ> * D * 2 + ta_stages<D, NQ> * ta_kb<NQ> * D * 2;

// floats of a part (one slice of one tile)
__host__ __device__ constexpr size_t ta_part_floats(int rows, int dim) { return (size_t) rows * (dim + 2); }

struct TaPlan
{
    amp_attention_args P;
    int nq;                                    // row tiles of 128 per CTA
    int tiles;                                 // row tiles per key-value head (an upper bound with cu)
    int slices;                                // of every tile's keys
    int split_rows;                            // sequences of up to so many rows (tokens x group) are the split form's
    int pdl;
    int group, each;                           // heads / kv_heads; tokens of every sequence without cu
    // what a CTA divides by before its first load (us with divisions / so: six prompts 33.6 / 32.5, six of 390 tokens in windows of 128 32.4 / 31.4);
    // tiles: of a sequence without cu
    AtDiv by_group, by_kv, by_slices, by_tiles;
    float scale2;                              // scale * log2(e)
    size_t part_offset;                        // of the parts in the workspace
    AtPages g;
};

int attention_tc(TaPlan& S, cudaStream_t stream);               // (fills group and what is behind it in)

}  // namespace amp
