// Copies of rows between the sequences of a cache (cache_copy.cu).
#pragma once
#include "common.cuh"
#include "copy_plan.cuh"

// Where a sequence's rows are: row r of block h (a head) of plane p of sequence s is row_bytes bytes at
// base + p * plane_stride + s * seq_stride + h * block_stride + r * row_bytes.
struct CopyGeometry {
  void* base;
  long long plane_stride, seq_stride, block_stride;
  int planes, blocks;
  int row_bytes;              // multiple of 4
};

// Programs of copy_plan over one geometry, one launch where they fit.  `hi` / `lo` of the programs count rows of the geometry.
int arcb_launch_cache_copy(const CopyGeometry& g, const std::vector<CopyProgram>& programs, const std::vector<char>& serial, cudaStream_t stream);
constexpr int COPY_MAX_STEPS = 1900;      // launch parameters end at 32764 bytes
void arcb_count_launch(long long n);
