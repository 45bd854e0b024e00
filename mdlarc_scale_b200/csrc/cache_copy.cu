// Copies of rows between the sequences of a cache: forks of a sequence, reorderings of many, compactions.
//
// A thread owns places (plane, head, row, 16 bytes) and carries out a whole program of copy_plan.cuh for them: loads and
// stores of that place in one sequence after the other.  Copies never move a row to another place, so no thread touches what
// another one reads or writes, and the program's order alone makes every read see what was there before the call: no barrier,
// no second buffer, and a source is read once however many sequences it goes to.  Programs come as launch parameters, which
// keeps the call free of device memory of its own (and a captured one independent of later calls).
#include "../../include/arcb200.h"
#include "cache_copy.cuh"
#include "launch.cuh"

int arcb_fail(int code, const char* msg);
int arcb_fail_cuda(cudaError_t e, const char* where);

namespace {

constexpr int CC_THREADS = 256;
constexpr int CC_UNROLL = 4;

template <int STEPS>
struct CopyArgs {
  CopyGeometry g;
  int n_programs, row_vecs;
  CopyStep step[STEPS];
  // of each program: first step and rows, packed where there is room for as many programs as steps / 2
  unsigned short first[STEPS / 2 + 1];
};

template <int STEPS, typename VEC>
__global__ void __launch_bounds__(CC_THREADS)
cache_copy_kernel(const __grid_constant__ CopyArgs<STEPS> a) {
  pdl_launch_dependents();
  pdl_wait();
  const int from = a.first[blockIdx.y], to = a.first[blockIdx.y + 1];
  // the first step is a load: its unused row fields hold the program's rows
  const int lo = a.step[from].begin, hi = a.step[from].end;
  const unsigned run = (unsigned)(hi - lo) * a.row_vecs;
  const unsigned total = run * (unsigned)(a.g.planes * a.g.blocks);
  const unsigned base = blockIdx.x * (unsigned)(CC_THREADS * CC_UNROLL);
  if (base >= total) return;
  char* at[CC_UNROLL];
  int row[CC_UNROLL];
#pragma unroll
  for (int u = 0; u < CC_UNROLL; ++u) {
    const unsigned i = base + u * CC_THREADS + threadIdx.x;
    const unsigned pb = i / run, off = i - pb * run;
    const unsigned p = pb / a.g.blocks, b = pb - p * a.g.blocks;
    row[u] = i < total ? lo + (int)(off / a.row_vecs) : -1;        // -1: no step has it
    at[u] = reinterpret_cast<char*>(a.g.base) + (i < total ? p * a.g.plane_stride + b * a.g.block_stride +
                                                             ((long long)lo * a.row_vecs + off) * (long long)sizeof(VEC) : 0);
  }
  VEC v[CC_UNROLL], held[CC_UNROLL];
  for (int s = from; s < to; ++s) {
    const CopyStep c = a.step[s];
    const long long d = c.slot * a.g.seq_stride;
    if (c.op == COPY_LOAD) {
#pragma unroll
      for (int u = 0; u < CC_UNROLL; ++u)
        if (row[u] >= 0) v[u] = *reinterpret_cast<const VEC*>(at[u] + d);
    } else if (c.op == COPY_STORE) {
#pragma unroll
      for (int u = 0; u < CC_UNROLL; ++u)
        if (row[u] >= c.begin && row[u] < c.end) *reinterpret_cast<VEC*>(at[u] + d) = v[u];
    } else if (c.op == COPY_HOLD) {
#pragma unroll
      for (int u = 0; u < CC_UNROLL; ++u)
        if (row[u] >= 0) held[u] = *reinterpret_cast<const VEC*>(at[u] + d);
    } else {
#pragma unroll
      for (int u = 0; u < CC_UNROLL; ++u)
        if (row[u] >= c.begin && row[u] < c.end) *reinterpret_cast<VEC*>(at[u] + d) = held[u];
    }
  }
}

template <int STEPS, typename VEC>
int launch_programs(const CopyGeometry& g, const CopyProgram* const* progs, int n, cudaStream_t stream) {
  CopyArgs<STEPS> a;
  a.row_vecs = g.row_bytes / (int)sizeof(VEC);
  a.n_programs = n;
  int steps = 0, rows = 0;
  for (int i = 0; i < n; ++i) {
    const CopyProgram& p = *progs[i];
    a.first[i] = (unsigned short)steps;
    for (size_t s = 0; s < p.steps.size(); ++s) a.step[steps + s] = p.steps[s];
    a.step[steps].begin = p.lo;
    a.step[steps].end = p.hi;
    steps += (int)p.steps.size();
    rows = p.hi - p.lo > rows ? p.hi - p.lo : rows;
  }
  a.first[n] = (unsigned short)steps;
  // places are numbered in 32 bits: a launch takes as many planes as that allows
  const long long per_plane = (long long)rows * a.row_vecs * g.blocks;
  if (per_plane > 0x7fffffffLL) return -1;
  const int at_once = (int)(0x7fffffffLL / per_plane);
  for (int p = 0; p < g.planes; p += at_once) {
    a.g = g;
    a.g.base = reinterpret_cast<char*>(g.base) + p * g.plane_stride;
    a.g.planes = g.planes - p < at_once ? g.planes - p : at_once;
    const long long places = per_plane * a.g.planes;
    const unsigned blocks = (unsigned)((places + CC_THREADS * CC_UNROLL - 1) / (CC_THREADS * CC_UNROLL));
    const cudaError_t e = arcb_launch(cache_copy_kernel<STEPS, VEC>, dim3(blocks, n), dim3(CC_THREADS), 0, stream, a);
    arcb_count_launch(1);
    if (e != cudaSuccess) return (int)e;
  }
  return 0;
}

template <typename VEC>
int launch_batch(const CopyGeometry& g, const std::vector<const CopyProgram*>& batch, size_t steps, cudaStream_t stream) {
  const int n = (int)batch.size();
  if (!n) return 0;
  if (steps <= 48) return launch_programs<48, VEC>(g, batch.data(), n, stream);
  if (steps <= 400) return launch_programs<400, VEC>(g, batch.data(), n, stream);
  return launch_programs<COPY_MAX_STEPS, VEC>(g, batch.data(), n, stream);
}

static_assert(sizeof(CopyArgs<COPY_MAX_STEPS>) <= 32764, "launch parameters");

}  // namespace

int arcb_launch_cache_copy(const CopyGeometry& g, const std::vector<CopyProgram>& programs, const std::vector<char>& serial, cudaStream_t stream) {
  const long long any = reinterpret_cast<long long>(g.base) | g.plane_stride | g.seq_stride | g.block_stride | g.row_bytes;
  if (any & 3) return -1;
  const bool wide = !(any & 15);
  std::vector<const CopyProgram*> batch;
  size_t steps = 0;
  auto flush = [&]() {
    const int r = wide ? launch_batch<uint4>(g, batch, steps, stream) : launch_batch<uint32_t>(g, batch, steps, stream);
    batch.clear();
    steps = 0;
    return r;
  };
  for (size_t i = 0; i < programs.size(); ++i) {
    if (steps + programs[i].steps.size() > COPY_MAX_STEPS || serial[i]) {
      const int r = flush();
      if (r) return r;
    }
    batch.push_back(&programs[i]);
    steps += programs[i].steps.size();
  }
  return flush();
}

extern "C" int arcb_op_cache_copy(void* d_cache, int32_t n_planes, int32_t n_seqs, int32_t n_heads, int32_t t_max, int32_t row_bytes,
                                  const int32_t* h_copies, int32_t n_copies, void* stream) {
  if (!d_cache || (n_copies > 0 && !h_copies)) return arcb_fail(ARCB_E_ARG, "null copy argument");
  if (n_planes <= 0 || n_seqs <= 0 || n_heads <= 0 || t_max <= 0 || n_copies < 0) return arcb_fail(ARCB_E_ARG, "bad copy sizes");
  if (row_bytes <= 0 || row_bytes % 4 || reinterpret_cast<uintptr_t>(d_cache) % 4)
    return arcb_fail(ARCB_E_ARG, "cache rows are multiples of 4 bytes, aligned to them");
  std::vector<CopyProgram> programs;
  std::vector<char> serial;
  try {
    switch (copy_plan(h_copies, n_copies, n_seqs, t_max, COPY_MAX_STEPS, programs, serial)) {
      case COPY_PLAN_RANGE: return arcb_fail(ARCB_E_ARG, "a copy names a sequence or rows outside the cache");
      case COPY_PLAN_TWICE: return arcb_fail(ARCB_E_ARG, "a sequence is written by two copies");
      case COPY_PLAN_CYCLE: return arcb_fail(ARCB_E_UNSUPPORTED, "copies that form a cycle of more than 950 sequences are not implemented");
    }
    CopyGeometry g{};
    g.base = d_cache;
    g.block_stride = (long long)t_max * row_bytes;
    g.seq_stride = g.block_stride * n_heads;
    g.plane_stride = g.seq_stride * n_seqs;
    g.planes = n_planes; g.blocks = n_heads; g.row_bytes = row_bytes;
    const int r = arcb_launch_cache_copy(g, programs, serial, (cudaStream_t)stream);
    if (r > 0) return arcb_fail_cuda((cudaError_t)r, "cache copy");
    if (r < 0) return arcb_fail(ARCB_E_ARG, "a plane of the cache is too large");
  } catch (const std::bad_alloc&) {
    return arcb_fail(ARCB_E_STATE, "out of host memory");
  }
  return ARCB_OK;
}
