// Operations on the pages of a paged KV cache (include/qe_paged.h): free, extend, fork, compact, copy.
//
// The allocation (table, ref) is a few hundred kilobytes at most, so what has to be decided in one order
// (which page goes to whom) is decided by one workgroup: ranks by ballots, free pages by a scan of ref that
// stops when enough are found. Everything else (releasing, sharing, renaming entries, moving data) is
// order-free and spread over the card; the counts are atomics whose sum does not depend on their order.
// Data moves in 32 KB pieces, eight 16-byte loads in flight per thread.
#include <algorithm>

#include "qe_device.hpp"
#include "qe_paged.h"

namespace qe {
namespace pages {

constexpr int PT = 1024;            // threads of the deciding workgroup
constexpr int PW = PT / WAVE;
constexpr int SCAN = 16;            // refs per thread and scan step
constexpr int WS_HEAD = 8;          // workspace: [0] pairs to move; from WS_HEAD on their pages

__device__ __forceinline__ bool valid(int id, int n) { return (unsigned)id < (unsigned)n; }

// Rank of this thread's flag among the block's true ones, in thread order, and their number. Two barriers.
struct Ranks {
  int rank, total;
};
__device__ __forceinline__ Ranks rank_of(bool f, int (&part)[PW]) {
  const unsigned long long m = __ballot(f);
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  __syncthreads();  // earlier reads of part are done
  if (lane == 0) part[w] = __popcll(m);
  __syncthreads();
  Ranks r{(int)__popcll(m & ((1ull << lane) - 1)), 0};
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    if (i < w) r.rank += part[i];
    r.total += part[i];
  }
  return r;
}

// The next `want` (<= PT) free ids from `at` on, ascending, into list; returns how many there were and moves
// `at` past the last one taken. ref <= 0 is free. Called by the whole block.
__device__ __forceinline__ int take_free(const int* ref, int N, int want, int& at, int* list,
                                         int (&part)[PW], int& next) {
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE;
  int got = 0;
  while (got < want && at < N) {
    unsigned long long m[SCAN];
    int mine = 0;
    const int base = at + w * (WAVE * SCAN);
#pragma unroll
    for (int i = 0; i < SCAN; ++i) {
      const int id = base + i * WAVE + lane;
      const int r = id < N ? ref[id] : 1;
      m[i] = __ballot(r <= 0);
      mine += __popcll(m[i]);
    }
    __syncthreads();  // earlier reads of part, list and next are done
    if (lane == 0) part[w] = mine;
    if (threadIdx.x == 0) next = at + PT * SCAN;
    __syncthreads();
    int rank = got, total = 0;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      if (i < w) rank += part[i];
      total += part[i];
    }
#pragma unroll
    for (int i = 0; i < SCAN; ++i) {
      const int r = rank + (int)__popcll(m[i] & ((1ull << lane) - 1));
      if ((m[i] >> lane & 1) && r < want) {
        const int id = base + i * WAVE + lane;
        list[r] = id;
        if (r == want - 1) next = id + 1;
      }
      rank += __popcll(m[i]);
    }
    __syncthreads();
    got = min(want, got + total);
    at = next;
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
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), w = tid / WAVE;
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
  if (lane == WAVE - 1) part[w] = s;
  __syncthreads();
  int C = 0;
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    if (i < w) s += part[i];
    C += part[i];
  }
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
    const int got = take_free(ref, N, r.total, at, list, part, next);
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

__global__ void __launch_bounds__(256)
fork_share_kernel(int* __restrict__ table, long ldt, int* __restrict__ ref, const int* __restrict__ src,
                  const int* __restrict__ dst, const int* __restrict__ length, int m, int B, int M, int N,
                  int lp) {
  __shared__ Pairs pairs;
  mark_pairs(pairs, src, dst, m, B);
  const int a = src[blockIdx.x], b = dst[blockIdx.x];
  if (refused(pairs, a, b, B)) return;
  const int whole = max(length[blockIdx.x], 0) >> lp;
  for (int j = blockIdx.y * 256 + threadIdx.x; j < M; j += gridDim.y * 256) {
    int* e = table + (size_t)b * ldt + j;
    const int old = *e;
    int id = j < whole ? table[(size_t)a * ldt + j] : -1;
    if (!valid(id, N)) id = -1;
    if (valid(old, N)) atomicSub(ref + old, 1);
    if (id >= 0) atomicAdd(ref + id, 1);
    if (id != old) *e = id;
  }
}

__global__ void __launch_bounds__(PT)
fork_tail_kernel(int* __restrict__ table, long ldt, int* __restrict__ ref, const int* __restrict__ src,
                 const int* __restrict__ dst, const int* __restrict__ length, int m,
                 int* __restrict__ missing, int* __restrict__ ws, int B, int M, int N, int lp) {
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
      from = table[(size_t)a * ldt + j];
      e = table + (size_t)b * ldt + j;
      need = valid(from, N);
    }
  }
  const int bad = rank_of(no, part).total;
  const Ranks r = rank_of(need, part);
  int at = 0;
  const int got = take_free(ref, N, r.total, at, list, part, next);
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
  __shared__ int part[PW], part2[PW];
  const int tid = threadIdx.x, lane = tid & (WAVE - 1), w = tid / WAVE;
  int* from = ws + WS_HEAD;
  int* into = from + N / 2;
  int* to = into + N / 2;
  int used = 0;
  for (int i = tid; i < N; i += PT) used += ref[i] > 0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) used += __shfl_xor(used, o);
  if (lane == 0) part[w] = used;
  __syncthreads();
  int U = 0;
#pragma unroll
  for (int i = 0; i < PW; ++i) U += part[i];
  int nf = 0, nu = 0;  // free ids below U, used ids from U on, so far
  for (int at = 0; at < N; at += PT * SCAN) {
    unsigned long long mf[SCAN], mu[SCAN];
    int cf = 0, cu = 0;
    const int base = at + w * (WAVE * SCAN);
#pragma unroll
    for (int i = 0; i < SCAN; ++i) {
      const int id = base + i * WAVE + lane;
      const bool in = id < N, full = in && ref[id] > 0;
      mf[i] = __ballot(in && !full && id < U);
      mu[i] = __ballot(full && id >= U);
      if (in && !full && id >= U) to[id] = id;
      cf += __popcll(mf[i]);
      cu += __popcll(mu[i]);
    }
    __syncthreads();
    if (lane == 0) part[w] = cf, part2[w] = cu;
    __syncthreads();
    int rf = nf, ru = nu;
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      if (i < w) rf += part[i], ru += part2[i];
      nf += part[i], nu += part2[i];
    }
    const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
    for (int i = 0; i < SCAN; ++i) {
      const int id = base + i * WAVE + lane;
      if (mf[i] >> lane & 1) into[rf + __popcll(mf[i] & below)] = id;
      if (mu[i] >> lane & 1) from[ru + __popcll(mu[i] & below)] = id;
      rf += __popcll(mf[i]);
      ru += __popcll(mu[i]);
    }
  }
  __threadfence_block();
  __syncthreads();
  for (int r = tid; r < nu; r += PT) {
    const int a = from[r], b = into[r];
    to[a] = b;
    ref[b] = ref[a];
    ref[a] = 0;
  }
  if (tid == 0) ws[0] = nu, ws[1] = U;
}

__global__ void __launch_bounds__(256)
compact_table_kernel(int* __restrict__ table, long ldt, const int* __restrict__ ws, int M, int N) {
  const int U = ws[1];
  const int* to = ws + WS_HEAD + 2 * (N / 2);
  for (int j = blockIdx.y * 256 + threadIdx.x; j < M; j += gridDim.y * 256) {
    int* e = table + (size_t)blockIdx.x * ldt + j;
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
};
// CHECK: the caller's pairs (see qe_kv_pages_copy); otherwise lists of this file, whose pages are in range
// and where no page is both source and destination.
template <bool CHECK>
__global__ void __launch_bounds__(CT) move_kernel(Move a) {
  const int m = a.count ? min(*a.count, a.m) : a.m;
  for (int r = blockIdx.x; r < m; r += gridDim.x) {
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
                              hipStream_t stream) {
  Move a{};
  a.pool[0] = static_cast<char*>(kp), a.pool[1] = static_cast<char*>(vp);
  a.page = page_bytes, a.layer = page_bytes * (size_t)N;
  a.pieces = (int)((page_bytes + PIECE - 1) / PIECE), a.units = layers * 2 * a.pieces, a.N = N;
  a.src = src, a.dst = dst, a.count = count, a.m = m;
  const int want = 8 * compute_units();  // workgroups: 8 pieces in flight per compute unit
  const int gx = std::min(m, want), gy = std::max(1, std::min({a.units, want / gx, 65535}));
  if (check)
    move_kernel<true><<<dim3(gx, gy), dim3(CT), 0, stream>>>(a);
  else
    move_kernel<false><<<dim3(gx, gy), dim3(CT), 0, stream>>>(a);
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
  pages::fork_share_kernel<<<pages::entry_grid(m, M), dim3(256), 0, stream>>>(table, ldt, ref, src, dst,
                                                                             length, m, B, M, N, lp);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  pages::fork_tail_kernel<<<dim3(1), dim3(pages::PT), 0, stream>>>(table, ldt, ref, src, dst, length, m,
                                                                  missing, w, B, M, N, lp);
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
  pages::compact_table_kernel<<<pages::entry_grid(B, M), dim3(256), 0, stream>>>(table, ldt, w, M, N);
  e = hipGetLastError();
  if (e != hipSuccess || N < 2) return e;
  return pages::launch_move(false, kp, vp, layers, page_bytes, w + pages::WS_HEAD,
                            w + pages::WS_HEAD + N / 2, w, N / 2, N, stream);
}

extern "C" hipError_t qe_kv_pages_copy(void* kp, void* vp, int layers, size_t page_bytes, const int* src,
                                       const int* dst, int m, int N, hipStream_t stream) {
  if (!pages::pool_ok(kp, vp, layers, page_bytes, N) || m < 1 || m > 65535 || !src || !dst)
    return hipErrorInvalidValue;
  return pages::launch_move(true, kp, vp, layers, page_bytes, src, dst, nullptr, m, N, stream);
}
