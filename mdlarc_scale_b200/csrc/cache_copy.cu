// Copies of rows between the sequences of a cache: forks of a sequence, reorderings of many, compactions.
//
// A thread owns places (plane, head, row, 16 bytes) and carries out a whole program of copy_plan.cuh for them: loads and
// stores of that place in one sequence after the other.  Copies never move a row to another place, so no thread touches what
// another one reads or writes, and the program's order alone makes every read see what was there before the call: no barrier,
// no second buffer, and a source is read once however many sequences it goes to.  Programs come as launch parameters, which
// keeps the call free of device memory of its own (and a captured one independent of later calls).
#include "../../include/arcb200.h"
#include "cache_copy.cuh"
#include "gemm.cuh"
#include "launch.cuh"

int arcb_fail(int code, const char* msg);
int arcb_fail_cuda(cudaError_t e, const char* where);

namespace {

constexpr int CC_THREADS = 256;

template <int STEPS>
struct CopyArgs {
  CopyGeometry g;
  int row_vecs, turns;        // vectors of a row; times that a CTA goes on by its threads' places
  CopyStep step[STEPS];
  unsigned short first[STEPS / 2 + 1];      // step of each program (which has two at least)
};

// place i of a program: its address in a sequence at 0, and its row (-1: there is none)
struct CopyPlace {
  char* at;
  int row;
};
template <typename VEC, int STEPS>
__device__ __forceinline__ CopyPlace cc_place(const CopyArgs<STEPS>& a, unsigned i, unsigned total, unsigned run, int lo) {
  CopyPlace p;
  const unsigned pb = i / run, off = i - pb * run, plane = pb / a.g.blocks, b = pb - plane * a.g.blocks;
  p.row = i < total ? lo + (int)(off / a.row_vecs) : -1;
  p.at = reinterpret_cast<char*>(a.g.base) + plane * a.g.plane_stride + b * a.g.block_stride + ((long long)lo * a.row_vecs + off) * (long long)sizeof(VEC);
  return p;
}

// Programs of one source: four places a thread in a turn, the next turn's rows on their way while this one's are written.  (A CTA a
// turn spent most of its time starting: 77 sequences moved in 475 us,
// now 436, 6.0 TB/s; 775 with the registers of the other kernel.)
template <int STEPS, typename VEC>
__global__ void __launch_bounds__(CC_THREADS)
cache_spread_kernel(const __grid_constant__ CopyArgs<STEPS> a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int U = 4;
  const int from = a.first[blockIdx.y], to = a.first[blockIdx.y + 1];
  // the first step is a load: its unused row fields hold the program's rows
  const int lo = a.step[from].begin, hi = a.step[from].end;
  const unsigned run = (unsigned)(hi - lo) * a.row_vecs, total = run * (unsigned)(a.g.planes * a.g.blocks);
  const long long src = a.step[from].slot * a.g.seq_stride;
  unsigned base = blockIdx.x * (unsigned)(CC_THREADS * U) * a.turns;
  if (base >= total) return;
  CopyPlace now[U], next[U];
  VEC v[U], w[U];
  auto fetch = [&](CopyPlace (&p)[U], VEC (&x)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      p[u] = cc_place<VEC>(a, base + u * CC_THREADS + threadIdx.x, total, run, lo);
      if (p[u].row >= 0) x[u] = *reinterpret_cast<const VEC*>(p[u].at + src);
    }
    base += CC_THREADS * U;
  };
  fetch(now, v);
  for (int t = 1;; ++t) {
    const bool more = t < a.turns && base < total;
    if (more) fetch(next, w);
    for (int s = from + 1; s < to; ++s) {
      const CopyStep c = a.step[s];
      const long long d = c.slot * a.g.seq_stride;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (now[u].row >= c.begin && now[u].row < c.end) *reinterpret_cast<VEC*>(now[u].at + d) = v[u];
    }
    if (!more) break;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      now[u] = next[u];
      v[u] = w[u];
    }
  }
}

// Programs of several sources: one place a thread.
template <int STEPS, typename VEC>
__global__ void __launch_bounds__(CC_THREADS)
cache_permute_kernel(const __grid_constant__ CopyArgs<STEPS> a) {
  pdl_launch_dependents();
  pdl_wait();
  const int from = a.first[blockIdx.y], to = a.first[blockIdx.y + 1];
  const int lo = a.step[from].begin, hi = a.step[from].end;
  const unsigned run = (unsigned)(hi - lo) * a.row_vecs, total = run * (unsigned)(a.g.planes * a.g.blocks), i = blockIdx.x * CC_THREADS + threadIdx.x;
  if (i >= total) return;
  const CopyPlace p = cc_place<VEC>(a, i, total, run, lo);
  VEC v[COPY_VALUES + 1];
  for (int s = from; s < to; ++s) {
    const CopyStep c = a.step[s];
    VEC* at = reinterpret_cast<VEC*>(p.at + c.slot * a.g.seq_stride);
    const bool mine = p.row >= c.begin && p.row < c.end;
#pragma unroll
    for (int k = 0; k <= COPY_VALUES; ++k) {       // one of them, the same for all threads
      if (c.op == k) v[k] = *at;
      else if (c.op == COPY_STORE + k && mine) *at = v[k];
    }
  }
}

template <int STEPS, typename VEC>
int launch_programs(const CopyGeometry& g, const std::vector<const CopyProgram*>& progs, bool single, cudaStream_t stream) {
  CopyArgs<STEPS> a;
  a.row_vecs = g.row_bytes / (int)sizeof(VEC);
  const int n = (int)progs.size();
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
    // up to eight turns, as long as sixteen CTAs an SM are left; one where a place is written many times anyway
    const long long turn = single ? CC_THREADS * 4 : CC_THREADS, ctas = (places + turn - 1) / turn * n;
    a.turns = !single || steps > 4 * n ? 1 : (int)(ctas >= 128LL * arcb_num_sms() ? 8 : ctas >= 32LL * arcb_num_sms() ? 2 : 1);
    const dim3 grid((unsigned)((places + turn * a.turns - 1) / (turn * a.turns)), n);
    const cudaError_t e = single ? arcb_launch(cache_spread_kernel<STEPS, VEC>, grid, dim3(CC_THREADS), 0, stream, a)
                                 : arcb_launch(cache_permute_kernel<STEPS, VEC>, grid, dim3(CC_THREADS), 0, stream, a);
    arcb_count_launch(1);
    if (e != cudaSuccess) return (int)e;
  }
  return 0;
}

template <typename VEC>
int launch_batch(const CopyGeometry& g, const std::vector<const CopyProgram*>& batch, size_t steps, bool single, cudaStream_t stream) {
  if (batch.empty()) return 0;
  if (steps <= 48) return launch_programs<48, VEC>(g, batch, single, stream);
  if (steps <= 400) return launch_programs<400, VEC>(g, batch, single, stream);
  return launch_programs<COPY_MAX_STEPS, VEC>(g, batch, single, stream);
}

static_assert(sizeof(CopyArgs<COPY_MAX_STEPS>) <= 32764, "launch parameters");

}  // namespace

int arcb_launch_cache_copy(const CopyGeometry& g, const std::vector<CopyProgram>& programs, const std::vector<char>& serial, cudaStream_t stream) {
  const long long any = reinterpret_cast<long long>(g.base) | g.plane_stride | g.seq_stride | g.block_stride | g.row_bytes;
  if (any & 3) return -1;
  const bool wide = !(any & 15);
  bool single = true;                      // every program has one source
  for (const CopyProgram& p : programs) {
    single = single && p.steps[0].op == 0;
    for (size_t s = 1; s < p.steps.size() && single; ++s) single = p.steps[s].op == COPY_STORE;
  }
  std::vector<const CopyProgram*> batch;
  size_t steps = 0;
  auto flush = [&]() {
    const int r = wide ? launch_batch<uint4>(g, batch, steps, single, stream) : launch_batch<uint32_t>(g, batch, steps, single, stream);
    batch.clear();
    steps = 0;
    return r;
  };
  for (size_t i = 0; i < programs.size(); ++i) {
    if (serial[i] || steps + programs[i].steps.size() > COPY_MAX_STEPS)
      if (const int r = flush()) return r;
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
