// Partial rows of a unit that several CTAs share (tree_attn.cu, tree_mma.cu). A CTA keeps up to two:
// slot 0 of a unit that an earlier CTA began, slot 1 of one that it begins and hands on. A slot:
//   float4 [head_dim / 4][block_rows]   O, unnormalised, of scale e^-m (rows innermost: a thread
//                                       per row writes, and the join reads, whole lines)
//   float  [block_rows]                 m, the maximum of the unscaled scores (or a bound within 2^8)
//   float  [block_rows]                 l
// The workspace is the error word (256 bytes) and the slots of every CTA.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

namespace jinf {

constexpr size_t TREE_WS_HEAD = 256;

__host__ __device__ __forceinline__ size_t part_floats(int block_rows, int hd) {
    return ((size_t)block_rows * (hd + 2) + 3) & ~(size_t)3;  // slots start on 16 bytes
}

struct TreeParams;
struct TreePlan;
cudaError_t tree_mma_launch(const TreeParams& p, const TreePlan& plan, bool bf, int head_dim, uint16_t* out, float* lse,
                            float* parts, int* err, cudaStream_t s);

}  // namespace jinf
