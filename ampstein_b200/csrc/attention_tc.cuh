// Launch interface of the prompt form of the attention (attention_tc.cu)
#pragma once
#include "attention.cuh"

namespace amp {

template <int D> constexpr int ta_nq = D <= 128 ? 2 : 1;       // tiles of 128 rows per CTA
template <int D> constexpr int ta_kb = D <= 128 ? 128 : 64;    // keys per tile
template <int D> constexpr int ta_stages = D == 64 ? 8 : 5;    // tiles of keys or values in shared memory
template <int D> constexpr int ta_threads = 128 * (ta_nq<D> + 1);
template <int D> constexpr int ta_smem = ta_nq<D> * 128 * D * 2 + ta_stages<D> * ta_kb<D> * D * 2;

// Tiles of rows that cover `rows` rows; floats of a part (one slice of one tile)
__host__ __device__ constexpr int ta_rows(int dim) { return dim <= 128 ? 256 : 128; }
__host__ __device__ constexpr size_t ta_part_floats(int dim) { return (size_t) ta_rows(dim) * (dim + 2); }

struct TaPlan
{
    amp_attention_args P;
    int tiles;                                 // row tiles per key-value head (an upper bound with cu)
    int slices;                                // of every tile's keys
    int split_rows;                            // sequences of up to so many rows (tokens x group) are the split form's
    int pdl;
    float scale2;                              // scale * log2(e)
    size_t part_offset;                        // of the parts in the workspace
    AtPages g;
};

int attention_tc(const TaPlan& S, cudaStream_t stream);

}  // namespace amp
