// Operations on the pages of a paged KV cache (include/qe_paged.h): free, extend, fork, compact, copy.
//
// The allocation (table, ref) is a few hundred kilobytes at most, so what has to be decided in one order
// (which page goes to whom) is decided by one workgroup: ranks by ballots, free pages by a scan of ref that
// stops when enough are found. Everything else (releasing, sharing, renaming entries, moving data) is
// order-free and spread over the card; the counts are atomics whose sum does not depend on their order.
// Data moves in 32 KB pieces, eight 16-byte loads in flight per thread, at 5.0 TB/s read and written (a copy of
// 1 GiB: 5.2). In a graph, compacting 500 pages (524 MB) takes 110 us, a fork of eight sequences in 8 layers (33.6 MB)
// 13.4, a free and an extend between two steps of 200 sequences 6.8: chains of loads, in one launch each. The fork's
// deciding workgroup (8.8 us, against 5 for extend's) reads the pairs three times and starts its scan behind a fence.
// A copy of the caller's pairs checks every pair against all others in every workgroup that moves a piece of it: of
// pages of 8 KB, 1,000 move at 3.9 TB/s and 30,000 at 1.7.
#include <algorithm>
#include <type_traits>

#include "qe_device.hpp"
#include "qe_paged.h"

namespace qe {
namespace pages {

constexpr int PT = 1024;            // threads of the deciding workgroup
constexpr int PW = PT / WAVE;
// Refs per thread and scan step: few in the first one, which nearly always finds what a call needs (a step of 16
// everywhere: extend 8.1 us against 3.2, compact's plan 8.1 against 2.4, since one compute unit runs all 16 waves
// of it), more in those after it.
constexpr int FEW = 2, MANY = 16;
constexpr int WS_HEAD = 8;          // workspace: [0] pairs to move; from WS_HEAD on their pages

__device__ __forceinline__ bool valid(int id, int n) { return (unsigned)id < (unsigned)n; }

// A step of the scan for free pages (ref <= 0): ids at .. at + PT * S - 1, a wave's WAVE * S of them in
// ballots. Agent-scope loads: the counts may have been changed by atomics of this kernel.
template <int S>
struct Step {
  unsigned long long m[S];
  int base, mine;
};
template <int S>
__device__ __forceinline__ Step<S> scan_step(const int* ref, int N, int at) {
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  Step<S> s;
  s.base = at + w * (WAVE * S);
  s.mine = 0;
  int r[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int id = s.base + i * WAVE + lane;
    r[i] = id < N ? __hip_atomic_load(ref + id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 1;
  }
#pragma unroll
  for (int i = 0; i < S; ++i) {
    s.m[i] = __ballot(r[i] <= 0);
    s.mine += __popcll(s.m[i]);
  }
  return s;
}

// Sums over the waves of what lane 0 of each passes: before this wave, and all. Two barriers.
struct Sums {
  int before, all;
};
__device__ __forceinline__ Sums wave_sums(int mine, int (&part)[PW]) {
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  __syncthreads();  // earlier reads of part are done
  if (lane == 0) part[w] = mine;
  __syncthreads();
  int v = lane < PW ? part[lane] : 0;
#pragma unroll
  for (int o = 1; o < PW; o <<= 1) {
    const int u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return Sums{w ? __builtin_amdgcn_readlane(v, __builtin_amdgcn_readfirstlane(w) - 1) : 0,
              __builtin_amdgcn_readlane(v, PW - 1)};
}

// Rank of this thread's flag among the block's true ones, in thread order, and their number.
struct Ranks {
  int rank, total;
};
__device__ __forceinline__ Ranks rank_of(bool f, int (&part)[PW]) {
  const unsigned long long m = __ballot(f);
  const Sums s = wave_sums(__popcll(m), part);
  return Ranks{s.before + (int)__popcll(m & ((1ull << (threadIdx.x & (WAVE - 1))) - 1)), s.all};
}

// The ids of a step from rank `got` on into list, up to `want` of them; next: one past the last taken.
template <int S>
__device__ __forceinline__ int take_step(const Step<S>& s, int got, int want, int at, int* list,
                                         int (&part)[PW], int& next) {
  const int lane = threadIdx.x & (WAVE - 1);
  const Sums t = wave_sums(s.mine, part);
  if (threadIdx.x == 0) next = at + PT * S;
  __syncthreads();
  int rank = got + t.before;
  if (rank < want) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int r = rank + (int)__popcll(s.m[i] & ((1ull << lane) - 1));
      if ((s.m[i] >> lane & 1) && r < want) {
        const int id = s.base + i * WAVE + lane;
        list[r] = id;
        if (r == want - 1) next = id + 1;
      }
      rank += __popcll(s.m[i]);
    }
  }
  __syncthreads();
  return min(want, got + t.all);
}

// The next `want` (<= PT) free ids from `at` on, ascending, into list; returns how many there were and moves
// `at` past the last one taken. Called by the whole block. first: a step at 0, loaded earlier.
__device__ __forceinline__ int take_free(const int* ref, int N, int want, int& at, int* list,
                                         int (&part)[PW], int& next, const Step<FEW>& first) {
  int got = 0;
  while (got < want && at < N) {
    got = at == 0 ? take_step(first, got, want, at, list, part, next)
                  : take_step(scan_step<MANY>(ref, N, at), got, want, at, list, part, next);
    at = next;
    __syncthreads();  // next is read before it is written again
  }
  return got;
}

// ---------------------------------------------------------------------------------- free
__global__ void __launch_bounds__(256)
free_kernel(int* __restrict__ table, long ldt, int* __restrict__ ref, const int* __restrict__ first,
            const int* __restrict__ last, int M, int N, int P) {
  const int b = blockIdx.x, f = first[b], l = last[b];
  for (int j = blockIdx.y * 256 + threadIdx.x; j < M; j += gridDim.y * 256) {
    if (j * P < f || (j + 1) * P > l) continue;  // M * P < 2^23
    int* e = table + (size_t)b * ldt + j;
    const int id = *e;
    if (valid(id, N)) atomicSub(ref + id, 1);
    if (id != -1) *e = -1;
  }
}

// ---------------------------------------------------------------------------------- extend
// Candidates: the entries of the pages in question, in (sequence, page) order, 1024 at a time.
__global__ void __launch_bounds__(PT)
extend_kernel(int* __restrict__ table, long ldt, int* __restrict__ ref, const int* __restrict__ pos,
              const int* __restrict__ count, int* __restrict__ missing, int B, int M, int N, int lp) {
  __shared__ int part[PW], list[PT], start[PT], first[PT], next;
  __shared__ unsigned long long over;
  const int tid = threadIdx.x, lane = tid & (WAVE - 1);
  const Step<FEW> ahead = scan_step<FEW>(ref, N, 0);  // beside the loads of the candidates
  if (tid == 0) over = 0;
  int n = 0;
  long long past = 0;
  if (tid < B) {
    const int p = pos[tid], c = count[tid];
    if (p >= 0 && c > 0) {
      const long long lo = p >> lp, hi = ((long long)p + c - 1) >> lp;
      first[tid] = (int)lo;
      n = (int)max(min(hi, (long long)M - 1) - lo + 1, 0ll);
      past = hi - lo + 1 - n;
    }
  }
  // inclusive sums of n over the sequences
  int s = n;
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const int v = __shfl_up(s, o);
    if (lane >= o) s += v;
  }
  const Sums sums = wave_sums(__builtin_amdgcn_readlane(s, WAVE - 1), part);
  s += sums.before;
  const int C = sums.all;
  start[tid] = s;  // candidates of sequences 0 .. tid
  if (past) atomicAdd(&over, (unsigned long long)past);
  __syncthreads();
  long long short_of = (long long)over;
  int at = 0;
  for (int x0 = 0; x0 < C; x0 += PT) {
    const int x = x0 + tid;
    int* e = nullptr;
    bool need = false;
    if (x < C) {
      int b = 0;  // the first sequence with start > x
#pragma unroll
      for (int o = PT / 2; o > 0; o >>= 1)
        if (start[b + o - 1] <= x) b += o;
      const int j = first[b] + x - (b ? start[b - 1] : 0);
      e = table + (size_t)b * ldt + j;
      need = !valid(*e, N);
    }
    const Ranks r = rank_of(need, part);
    if (r.total == 0) continue;  // uniform
    const int got = take_free(ref, N, r.total, at, list, part, next, ahead);
    short_of += r.total - got;
    if (need && r.rank < got) {
      const int id = list[r.rank];
      *e = id;
      ref[id] = 1;
    }
  }
  if (tid == 0) *missing = (int)min(short_of, 0x7fffffffll);
}

// ---------------------------------------------------------------------------------- fork
// Which pairs are refused: flags of the sequences that are sources, and how often each is a dst.
struct Pairs {
  int dsts[QE_PAGED_MAX_SEQS];
  bool srcs[QE_PAGED_MAX_SEQS];
};
__device__ __forceinline__ void mark_pairs(Pairs& s, const int* src, const int* dst, int m, int B) {
  for (int i = threadIdx.x; i < QE_PAGED_MAX_SEQS; i += blockDim.x) s.dsts[i] = 0, s.srcs[i] = false;
  __syncthreads();
  for (int i = threadIdx.x; i < m; i += blockDim.x) {
    if (valid(src[i], B)) s.srcs[src[i]] = true;
    if (valid(dst[i], B)) atomicAdd(&s.dsts[dst[i]], 1);
  }
  __syncthreads();
}
__device__ __forceinline__ bool refused(const Pairs& s, int src, int dst, int B) {
  return !valid(src, B) || !valid(dst, B) || s.srcs[dst] || s.dsts[dst] > 1;
}

// Releases dst's entries and shares src's whole pages, for entry j of a pair.
__device__ __forceinline__ void share_entry(int* table, long ldt, int* ref, int a, int b, int whole, int j,
                                            int N) {
  int* e = table + (size_t)b * ldt + j;
  const int old = *e;
  int id = j < whole ? table[(size_t)a * ldt + j] : -1;
  if (!valid(id, N)) id = -1;
  if (valid(old, N)) atomicSub(ref + old, 1);
  if (id >= 0) atomicAdd(ref + id, 1);
  if (id != old) *e = id;
}
__global__ void __launch_bounds__(256)
fork_share_kernel(int* __restrict__ table, long ldt, int* __restrict__ ref, const int* __restrict__ src,
                  const int* __restrict__ dst, const int* __restrict__ length, int m, int B, int M, int N,
                  int lp) {
  __shared__ Pairs pairs;
  mark_pairs(pairs, src, dst, m, B);
  const int a = src[blockIdx.x], b = dst[blockIdx.x];
  if (refused(pairs, a, b, B)) return;
  const int whole = max(length[blockIdx.x], 0) >> lp;
  for (int j = blockIdx.y * 256 + threadIdx.x; j < M; j += gridDim.y * 256)
    share_entry(table, ldt, ref, a, b, whole, j, N);
}

// The partial pages. SHARE: fork_share_kernel's work first, by this workgroup (m * M entries).
constexpr int SHARE_MOST = 8 * PT;
template <bool SHARE>
__global__ void __launch_bounds__(PT)
fork_tail_kernel(int* table, long ldt, int* ref, const int* __restrict__ src, const int* __restrict__ dst,
                 const int* __restrict__ length, int m, int* __restrict__ missing, int* __restrict__ ws,
                 int B, int M, int N, int lp) {
  __shared__ Pairs pairs;
  __shared__ int part[PW], list[PT], next;
  mark_pairs(pairs, src, dst, m, B);
  const int i = threadIdx.x;
  bool no = false, need = false;
  int from = -1, *e = nullptr;
  if (i < m) {
    const int a = src[i], b = dst[i], len = max(length[i], 0), j = len >> lp;
    no = refused(pairs, a, b, B);
    if (!no && j < M && (len & ((1 << lp) - 1))) {
      from = table[(size_t)a * ldt + j];  // (sources are no destinations: not changed here)
      e = table + (size_t)b * ldt + j;
      need = valid(from, N);
    }
  }
  if constexpr (SHARE) {
    for (int x = threadIdx.x; x < m * M; x += PT) {
      const int k = x / M, a = src[k], b = dst[k];
      if (!refused(pairs, a, b, B))
        share_entry(table, ldt, ref, a, b, max(length[k], 0) >> lp, x - k * M, N);
    }
    __threadfence();
    __syncthreads();  // the counts are final, and the entries written, before the partial pages'
  }
  const Step<FEW> first = scan_step<FEW>(ref, N, 0);
  const int bad = rank_of(no, part).total;
  const Ranks r = rank_of(need, part);
  int at = 0;
  const int got = take_free(ref, N, r.total, at, list, part, next, first);
  if (need && r.rank < got) {
    const int id = list[r.rank];
    *e = id;
    ref[id] = 1;
    ws[WS_HEAD + r.rank] = from;
    ws[WS_HEAD + N + r.rank] = id;
  }
  if (i == 0) {
    *missing = bad + r.total - got;
    ws[0] = got;
  }
}

// ---------------------------------------------------------------------------------- compact
// Workspace: [0] the number of moves; their sources, N / 2; their destinations, N / 2; the new id of every
// id >= U, N.
__global__ void __launch_bounds__(PT)
compact_plan_kernel(int* __restrict__ ref, int* __restrict__ ws, int N) {
  constexpr int NEAR = 4096;  // moves kept in LDS for the last step
  __shared__ int part[PW], near_from[NEAR], near_into[NEAR];
  const int tid = threadIdx.x, lane = tid & (WAVE - 1);
  int* from = ws + WS_HEAD;
  int* into = from + N / 2;
  int* to = into + N / 2;
  const Step<FEW> first = scan_step<FEW>(ref, N, 0);  // (ballots of the free ids; N and above count as used)
  int used = 0;
  for (int i = min(N, PT * FEW) + tid; i < N; i += PT) used += ref[i] > 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) used += __shfl_xor(used, o);
  const int U = wave_sums(used + max(0, min(N - first.base, WAVE * FEW)) - first.mine, part).all;
  int nf = 0, nu = 0;  // free ids below U, used ids from U on, so far
  const auto lists = [&](const auto& s, auto size) __attribute__((always_inline)) {
    constexpr int S = decltype(size)::value;
    unsigned long long mf[S], mu[S];
    int cf = 0, cu = 0;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int id = s.base + i * WAVE + lane;
      const bool in = id < N, full = in && !(s.m[i] >> lane & 1);
      mf[i] = __ballot(in && !full && id < U);
      mu[i] = __ballot(full && id >= U);
      if (in && !full && id >= U) to[id] = id;
      cf += __popcll(mf[i]);
      cu += __popcll(mu[i]);
    }
    const Sums tf = wave_sums(cf, part), tu = wave_sums(cu, part);
    int rf = nf + tf.before, ru = nu + tu.before;
    nf += tf.all, nu += tu.all;
    const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int id = s.base + i * WAVE + lane;
      if (mf[i] >> lane & 1) {
        const int r = rf + __popcll(mf[i] & below);
        into[r] = id;
        if (r < NEAR) near_into[r] = id;
      }
      if (mu[i] >> lane & 1) {
        const int r = ru + __popcll(mu[i] & below);
        from[r] = id;
        if (r < NEAR) near_from[r] = id;
      }
      rf += __popcll(mf[i]);
      ru += __popcll(mu[i]);
    }
  };
  lists(first, std::integral_constant<int, FEW>{});
  for (int at = PT * FEW; at < N; at += PT * MANY)
    lists(scan_step<MANY>(ref, N, at), std::integral_constant<int, MANY>{});
  __threadfence_block();
  __syncthreads();
  for (int r = tid; r < nu; r += PT) {
    const int a = r < NEAR ? near_from[r] : from[r], b = r < NEAR ? near_into[r] : into[r];
    to[a] = b;
    ref[b] = ref[a];
    ref[a] = 0;
  }
  if (tid == 0) ws[0] = nu, ws[1] = U;
}

__device__ __forceinline__ void compact_table(int* table, long ldt, const int* ws, int b, int j0, int dj, int M,
                                              int N) {
  const int U = ws[1];
  const int* to = ws + WS_HEAD + 2 * (N / 2);
  for (int j = j0; j < M; j += dj) {
    int* e = table + (size_t)b * ldt + j;
    const int id = *e;
    if (valid(id, N) && id >= U) *e = to[id];
  }
}

// ---------------------------------------------------------------------------------- data
constexpr int CT = 256, CU = 8, PIECE = CT * CU * 16;  // bytes of a piece: 32 KB

struct Move {
  char* pool[2];
  size_t page, layer;  // bytes
  int units, pieces, N;  // pieces of a page; units of a pair: layers * 2 * pieces
  const int *src, *dst, *count;  // count: device number of pairs (null: m)
  int m;
  int gx;                        // workgroups in x that move; further ones rename table entries (compact)
  int* table;
  const int* ws;
  long ldt;
  int M;
};
// CHECK: the caller's pairs (see qe_kv_pages_copy); otherwise lists of this file, whose pages are in range
// and where no page is both source and destination.
template <bool CHECK>
__global__ void __launch_bounds__(CT) move_kernel(Move a) {
  if ((int)blockIdx.x >= a.gx) {  // sequence blockIdx.x - gx
    compact_table(a.table, a.ldt, a.ws, blockIdx.x - a.gx, blockIdx.y * CT + threadIdx.x, gridDim.y * CT, a.M,
                  a.N);
    return;
  }
  const int m = a.count ? min(*a.count, a.m) : a.m;
  for (int r = blockIdx.x; r < m; r += a.gx) {
    const int s = a.src[r], d = a.dst[r];
    if constexpr (CHECK) {
      bool no = !valid(s, a.N) || !valid(d, a.N) || s == d;
      for (int i = threadIdx.x; i < m; i += CT) no |= a.src[i] == d || (i > r && a.dst[i] == d);
      if (__syncthreads_or(no)) continue;
    }
    for (int u = blockIdx.y; u < a.units; u += gridDim.y) {
      const int piece = u % a.pieces, lk = u / a.pieces;
      char* pool = a.pool[lk & 1] + (size_t)(lk >> 1) * a.layer + (size_t)piece * PIECE;
      const u32x4_t* from = reinterpret_cast<const u32x4_t*>(pool + (size_t)s * a.page) + threadIdx.x;
      u32x4_t* into = reinterpret_cast<u32x4_t*>(pool + (size_t)d * a.page) + threadIdx.x;
      const int left = (int)((min((size_t)PIECE, a.page - (size_t)piece * PIECE) / 16));
      u32x4_t x[CU];
#pragma unroll
      for (int i = 0; i < CU; ++i)
        if ((int)threadIdx.x + i * CT < left) x[i] = __builtin_nontemporal_load(from + i * CT);
#pragma unroll
      for (int i = 0; i < CU; ++i)
        if ((int)threadIdx.x + i * CT < left) __builtin_nontemporal_store(x[i], into + i * CT);
    }
  }
}

static bool pool_ok(const void* kp, const void* vp, int layers, size_t page_bytes, int N) {
  return kp && vp && ((reinterpret_cast<uintptr_t>(kp) | reinterpret_cast<uintptr_t>(vp)) & 15) == 0 &&
         layers >= 1 && layers <= 65535 && page_bytes >= 16 && page_bytes % 16 == 0 &&
         page_bytes <= (1u << 30) && N >= 1 && N <= (1 << 24) &&
         (size_t)layers * 2 * ((page_bytes + PIECE - 1) / PIECE) <= 0x7fffffff;
}
static bool alloc_ok(const void* table, long ldt, const void* ref, int B, int M, int N, int P) {
  return table && ref && B >= 1 && B <= QE_PAGED_MAX_SEQS && M >= 1 && ldt >= M && N >= 1 &&
         N <= (1 << 24) && P >= 16 && P <= 32768 && (P & (P - 1)) == 0 && (long)M * P <= (1 << 23) - 64;
}
static dim3 entry_grid(int rows, int M) { return dim3(rows, (unsigned)std::min((M + 255) / 256, 64)); }

static hipError_t launch_move(bool check, void* kp, void* vp, int layers, size_t page_bytes,
                              const int* src, const int* dst, const int* count, int m, int N,
                              hipStream_t stream, int* table = nullptr, long ldt = 0, const int* ws = nullptr,
                              int B = 0, int M = 0) {
  Move a{};
  a.pool[0] = static_cast<char*>(kp), a.pool[1] = static_cast<char*>(vp);
  a.page = page_bytes, a.layer = page_bytes * (size_t)N;
  a.pieces = (int)((page_bytes + PIECE - 1) / PIECE), a.units = layers * 2 * a.pieces, a.N = N;
  a.src = src, a.dst = dst, a.count = count, a.m = m;
  const int want = 8 * compute_units();  // workgroups: 8 pieces in flight per compute unit
  a.gx = std::min(m, want);
  const int gy = std::max(1, std::min({a.units, want / std::max(a.gx, 1), 65535}));
  a.table = table, a.ws = ws, a.ldt = ldt, a.M = M;
  const dim3 grid(a.gx + B, gy);
  if (check)
    move_kernel<true><<<grid, dim3(CT), 0, stream>>>(a);
  else
    move_kernel<false><<<grid, dim3(CT), 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace pages
}  // namespace qe

using namespace qe;

extern "C" hipError_t qe_kv_pages_free(int* table, long ldt, int* ref, const int* first,
                                       const int* last, int B, int M, int N, int P,
                                       hipStream_t stream) {
  if (!pages::alloc_ok(table, ldt, ref, B, M, N, P) || !first || !last) return hipErrorInvalidValue;
  pages::free_kernel<<<pages::entry_grid(B, M), dim3(256), 0, stream>>>(table, ldt, ref, first, last, M, N,
                                                                       P);
  return hipGetLastError();
}

extern "C" hipError_t qe_kv_pages_extend(int* table, long ldt, int* ref, const int* pos,
                                         const int* count, int* missing, int B, int M, int N, int P,
                                         hipStream_t stream) {
  if (!pages::alloc_ok(table, ldt, ref, B, M, N, P) || !pos || !count || !missing)
    return hipErrorInvalidValue;
  pages::extend_kernel<<<dim3(1), dim3(pages::PT), 0, stream>>>(table, ldt, ref, pos, count, missing, B, M,
                                                               N, __builtin_ctz((unsigned)P));
  return hipGetLastError();
}

extern "C" size_t qe_kv_pages_ws_size(int N) {
  return N < 1 ? 0 : (2 * (size_t)N + pages::WS_HEAD) * sizeof(int);
}

extern "C" hipError_t qe_kv_pages_fork(int* table, long ldt, int* ref, const int* src, const int* dst,
                                       const int* length, int m, void* kp, void* vp, int layers,
                                       size_t page_bytes, int* missing, void* ws, int B, int M, int N,
                                       int P, hipStream_t stream) {
  if (!pages::alloc_ok(table, ldt, ref, B, M, N, P) || !pages::pool_ok(kp, vp, layers, page_bytes, N) ||
      m < 1 || m > pages::PT || !src || !dst || !length || !missing || !ws ||
      (reinterpret_cast<uintptr_t>(ws) & 3))
    return hipErrorInvalidValue;
  const int lp = __builtin_ctz((unsigned)P);
  int* w = static_cast<int*>(ws);
  hipError_t e = hipSuccess;
  if ((long)m * M <= pages::SHARE_MOST) {
    pages::fork_tail_kernel<true><<<dim3(1), dim3(pages::PT), 0, stream>>>(table, ldt, ref, src, dst, length, m,
                                                                          missing, w, B, M, N, lp);
  } else {
    pages::fork_share_kernel<<<pages::entry_grid(m, M), dim3(256), 0, stream>>>(table, ldt, ref, src, dst,
                                                                               length, m, B, M, N, lp);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    pages::fork_tail_kernel<false><<<dim3(1), dim3(pages::PT), 0, stream>>>(table, ldt, ref, src, dst, length, m,
                                                                           missing, w, B, M, N, lp);
  }
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  return pages::launch_move(false, kp, vp, layers, page_bytes, w + pages::WS_HEAD, w + pages::WS_HEAD + N, w,
                            std::min(m, N), N, stream);
}

extern "C" hipError_t qe_kv_pages_compact(int* table, long ldt, int* ref, void* kp, void* vp, int layers,
                                          size_t page_bytes, void* ws, int B, int M, int N,
                                          hipStream_t stream) {
  if (!pages::alloc_ok(table, ldt, ref, B, M, N, 16) || !pages::pool_ok(kp, vp, layers, page_bytes, N) ||
      !ws || (reinterpret_cast<uintptr_t>(ws) & 3))
    return hipErrorInvalidValue;
  int* w = static_cast<int*>(ws);
  pages::compact_plan_kernel<<<dim3(1), dim3(pages::PT), 0, stream>>>(ref, w, N);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // (N = 1: nothing to move, no entry to rename)
  return pages::launch_move(false, kp, vp, layers, page_bytes, w + pages::WS_HEAD,
                            w + pages::WS_HEAD + N / 2, w, N / 2, N, stream, table, ldt, w, B, M);
}

extern "C" hipError_t qe_kv_pages_copy(void* kp, void* vp, int layers, size_t page_bytes, const int* src,
                                       const int* dst, int m, int N, hipStream_t stream) {
  if (!pages::pool_ok(kp, vp, layers, page_bytes, N) || m < 1 || m > 65535 || !src || !dst)
    return hipErrorInvalidValue;
  return pages::launch_move(true, kp, vp, layers, page_bytes, src, dst, nullptr, m, N, stream);
}
