// The paged K/V cache's bookkeeping and row moves: block tables and slots
// from request lengths, new rows into their slots, accepted rows of a
// drafted tree to the end of the context.  The attention that reads the
// cache is in tree.cu.
//
// A pool holds n_pages pages of page_size rows for each K/V head; request r
// keeps position t in page block_tables[r][t / page_size], row
// t % page_size, and slot = page * page_size + row names one row of every
// head.  Every page number and slot is checked against the pool before it
// is used as an address.
#include <algorithm>
#include <climits>
#include <mutex>

#include <cooperative_groups.h>

#include "halo_common.cuh"

namespace halo {

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);

namespace paged {

// ======================================================================
// tables_kernel: one launch, one cluster of 1 to 8 CTAs.
//
// Request r holds ceil(old/P) pages and is to hold ceil(new/P).  With g_r
// pages given back, n_r pages needed and their running sums G_r, N_r, the
// stack S is the free list followed by every page given back (request order,
// table order), and page k of the allocation order is S[have - 1 - k],
// have = n_free + G_R.  A request is granted if N_r <= have, so each page is
// found from two prefix sums and nothing is popped one at a time.
//
// Every CTA forms the prefix sums of all requests for itself (two passes of
// shuffles over shared memory; R is at most 8192) and takes a share of the new
// table entries, of the pages given back and, behind a cluster barrier, of the
// tokens, whose pages are then all in the tables.  n_free_out may alias n_free:
// it is written behind the same barrier.  A warp takes 32 consecutive pages or
// tokens: one search for all of them.  Latency-bound: a few integers a request
// and 16 B a token.  8 requests: 5.6 us on the device; 1024 requests with 42000
// new tokens: 15.4 us (22.5 us with a binary search a thread; 1.8 us each for
// the two passes over the requests, 1.7 us for the new entries, 4 us for the
// pages given back, 5 us for the tokens).
//
// STEP is a cache's next step: request r has a context of ctx rows, holds pages
// for old >= ctx of them (more than ctx where a step was given up) and is to
// hold ctx + max(count, 0).  Its new rows begin at ctx, in pages it holds
// already or takes.  The caller has packed its rows by the counts and does not
// know who is refused, so every request has its count's places in the slots,
// refused ones filled with -1.  old is updated in place: behind the cluster
// barrier, when every CTA has read it.
constexpr int kTabThreads = 1024;
constexpr int kTabMaxReq = 8192;
constexpr int kTabArrays = 7;      // shared int arrays of R entries

struct TablesParams {
  int32_t* table;
  int64_t table_stride;
  const int32_t* old_lens;
  const int32_t* new_lens;               // STEP: counts
  const int32_t* ctx;                    // STEP alone, as rows and held
  int32_t* rows;                         // new rows granted
  int32_t* starts;                       // places of its rows
  int32_t* held;                         // old_lens, to be updated
  int32_t* free_pages;
  const int32_t* n_free;
  int32_t* n_free_out;
  int64_t* slots;
  int64_t* positions;
  int32_t* cu;
  int32_t* lens;
  int32_t R, max_blocks, page, cap, T;
  uint32_t page_magic;                   // ceil(2^32 / page)
};

// Inclusive block scan of one 64-bit value a thread; *total gets the sum.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* s_warp, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();                       // s_warp is free again
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  int64_t w = s_warp[lane];              // kTabThreads / 32 == 32 warps
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, w, d);
    if (lane >= d) w += o;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int64_t before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
  return v + (warp > 0 ? before : 0);
}

// Pages of n rows (any value for a negative n, which is refused).
__device__ __forceinline__ int blocks(int n, int page) {
  const uint32_t b = (uint32_t)n / (uint32_t)page;
  return (int)(b + ((uint32_t)n - b * (uint32_t)page != 0 ? 1u : 0u));
}

// What request r has and wants: pages for `old` rows now and `want` rows then,
// new rows from `from` on.  False where that cannot be (a negative length, one
// that the table cannot hold): the request stays as it is.
template <bool STEP>
__device__ __forceinline__ bool load_lens(const TablesParams& p, int r, int& old, int& want,
                                          int& from) {
  old = p.old_lens[r];
  if constexpr (STEP) {
    from = p.ctx[r];
    const int64_t n = (int64_t)from + max(p.new_lens[r], 0);
    want = (int)min(n, (int64_t)INT_MAX);
    return from >= 0 && from <= old && blocks(old, p.page) <= p.max_blocks &&
           blocks(want, p.page) <= p.max_blocks;
  } else {
    from = old;
    want = p.new_lens[r];
    return old >= 0 && want >= 0 && blocks(old, p.page) <= p.max_blocks &&
           blocks(want, p.page) <= p.max_blocks;
  }
}

// First i in [0, n) with a[i] > k (running sums, k < a[n - 1]) for the warp's
// smallest k, found by all lanes together: 32 probes a step.
__device__ __forceinline__ int warp_find(const int32_t* a, int n, int k) {
  const int lane = threadIdx.x & 31;
  int lo = 0;
  while (n > 1) {
    const int step = n <= 32 ? 1 : (n + 31) >> 5 | 1;   // odd: 32 banks
    const int at = min((lane + 1) * step, n) - 1;
    const int f = __ffs(__ballot_sync(0xffffffffu, a[lo + at] > k)) - 1;
    lo += f * step;
    n = min(step, n - f * step);
  }
  return lo;
}

template <bool STEP>
__global__ void __launch_bounds__(kTabThreads) tables_kernel(const TablesParams p) {
  extern __shared__ int32_t sm[];
  __shared__ int64_t s_warp[32];
  __shared__ int s_used;
  int32_t* s_need = sm;                  // inclusive running sums
  int32_t* s_give = sm + p.R;
  int32_t* s_tok = sm + 2 * p.R;
  int32_t* s_old = sm + 3 * p.R;         // positions of its new rows: from, to
  int32_t* s_new = sm + 4 * p.R;
  int32_t* s_ob = sm + 5 * p.R;          // pages held before, and asked for
  int32_t* s_nb = sm + 6 * p.R;
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  const int n_cta = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int n_free = min(max(*p.n_free, 0), p.cap);
  if (threadIdx.x == 0) s_used = 0;

  // pass 1: pages needed and given back.  Both totals are at most
  // R * max_blocks < 2^31, so one 64-bit scan carries the two.
  int64_t carry = 0, total;
  for (int base = 0; base < p.R; base += kTabThreads) {
    const int r = base + threadIdx.x;
    int64_t v = 0;
    if (r < p.R) {
      int o, n, from;
      const bool ok = load_lens<STEP>(p, r, o, n, from);
      const int ob = blocks(o, p.page), nb = blocks(n, p.page);
      if (ok) v = nb > ob ? nb - ob : (int64_t)(ob - nb) << 32;
      s_old[r] = from;
      s_ob[r] = ob;
      s_nb[r] = nb;
      s_new[r] = ok ? n : from;
    }
    const int64_t s = carry + block_scan(v, s_warp, &total);
    carry += total;
    if (r < p.R) {
      s_need[r] = (int32_t)(s & 0xffffffff);
      s_give[r] = (int32_t)(s >> 32);
    }
  }
  const int n_give = (int)(carry >> 32);
  const int have = (int)min((int64_t)n_free + n_give, (int64_t)p.cap);
  __syncthreads();

  // pass 2: who is granted, and the running count of new tokens (STEP: of
  // those granted, and of those asked for, which the places go by)
  int64_t asked = 0;
  carry = 0;
  int used = 0;
  for (int base = 0; base < p.R; base += kTabThreads) {
    const int r = base + threadIdx.x;
    int64_t v = 0;
    if (r < p.R) {
      const bool needs = s_need[r] > (r > 0 ? s_need[r - 1] : 0);
      const bool granted = !needs || s_need[r] <= have;
      if (granted && needs) used = max(used, s_need[r]);
      if (!granted) s_new[r] = s_old[r];
      v = max(0, s_new[r] - s_old[r]);
    }
    const int64_t s = carry + block_scan(v, s_warp, &total);
    carry += total;
    if (r < p.R) {
      const int32_t c = (int32_t)min(s, (int64_t)INT_MAX);
      if constexpr (!STEP) s_tok[r] = c;
      if (rank == 0) {
        p.cu[r + 1] = c;
        if constexpr (STEP) p.rows[r] = (int32_t)v;
        else p.lens[r] = s_new[r];
      }
    }
    if constexpr (STEP) {
      const int64_t n = r < p.R ? max(p.new_lens[r], 0) : 0;
      const int64_t end = asked + block_scan(n, s_warp, &total);
      asked += total;
      if (r < p.R) {
        s_tok[r] = (int32_t)min(end, (int64_t)INT_MAX);
        if (rank == 0) p.starts[r] = (int32_t)min(end - n, (int64_t)INT_MAX);
      }
    }
  }
  if (used > 0) atomicMax(&s_used, used);
  __syncthreads();
  used = s_used;
  if (rank == 0 && threadIdx.x == 0) p.cu[0] = 0;
  const int n_tok = (int)min(STEP ? asked : carry, (int64_t)p.T);
  const int i0 = rank * kTabThreads + threadIdx.x, di = n_cta * kTabThreads;
  const int lane = threadIdx.x & 31;
  // Entry k of the stack: the free list, then the pages given back.  `low` is
  // the smallest k of the warp's lanes that ask (all lanes come here).
  auto stack = [&](int k, int low, bool ask) -> int32_t {
    int r = 0;
    if (__any_sync(0xffffffffu, ask && k >= n_free))
      r = warp_find(s_give, p.R, max(low - n_free, 0));
    if (!ask) return 0;
    if (k < n_free) return p.free_pages[k];
    const int g = k - n_free;
    while (g >= s_give[r]) ++r;
    return p.table[(int64_t)r * p.table_stride + s_nb[r] + (g - (r > 0 ? s_give[r - 1] : 0))];
  };

  // the new entries of the block tables
  for (int k0 = i0 - lane; k0 < used; k0 += di) {
    const int k = k0 + lane, last = min(k0 + 31, used - 1);
    const int32_t pg = stack(have - 1 - k, have - 1 - last, k < used);
    int r = warp_find(s_need, p.R, k0);
    if (k < used) {
      while (k >= s_need[r]) ++r;
      p.table[(int64_t)r * p.table_stride + s_ob[r] + (k - (r > 0 ? s_need[r - 1] : 0))] = pg;
    }
  }
  // pages given back that nobody took join the free list
  const int left = have - used;
  for (int k0 = n_free + i0 - lane; k0 < left; k0 += di) {
    const int k = k0 + lane;
    const int32_t pg = stack(k, k0, k < left);
    if (k < left) p.free_pages[k] = pg;
  }

  cl.sync();                             // all table entries are written, n_free was read
  if (rank == 0 && threadIdx.x == 0) *p.n_free_out = left;
  if constexpr (STEP) {
    for (int r = i0; r < p.R; r += di) {
      int o, n, from;
      if (!load_lens<STEP>(p, r, o, n, from)) continue;
      const bool needs = s_need[r] > (r > 0 ? s_need[r - 1] : 0);
      if (!needs || s_need[r] <= have) p.held[r] = n;
    }
  }

  // the slots of the new tokens (a row without a token gets -1), two of them
  // kTabThreads apart in flight
  for (int64_t t0 = i0 - lane; t0 < p.T; t0 += 2 * (int64_t)di) {
    int64_t slot[2];
    int pos[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t te = t0 + (int64_t)e * di;
      slot[e] = pos[e] = -1;
      if (te < n_tok) {                    // uniform in the warp
        int r = warp_find(s_tok, p.R, (int)te);
        const int t = (int)te + lane;
        if (t < n_tok) {
          while (t >= s_tok[r]) ++r;
          const int i = t - (r > 0 ? s_tok[r - 1] : 0);
          if (!STEP || i < s_new[r] - s_old[r]) {   // not one that was refused
            pos[e] = s_old[r] + i;
            int b = (int)__umulhi((uint32_t)pos[e], p.page_magic);   // exact or one more
            if (p.page == 1) b = pos[e];
            b -= (uint32_t)b * (uint32_t)p.page > (uint32_t)pos[e] ? 1 : 0;
            slot[e] = (int64_t)p.table[(int64_t)r * p.table_stride + b] * p.page +
                      (pos[e] - b * p.page);
          }
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t t = t0 + (int64_t)e * di + lane;
      if (t < p.T) {
        p.slots[t] = slot[e];
        p.positions[t] = pos[e];
      }
    }
  }
}

// ======================================================================
// Row copies.  A row of one head is D elements; VEC is the widest access
// that divides the row, every stride and every address.
struct Pool {
  char* k;
  char* v;
  int64_t k_sp, k_sh, k_st, v_sp, v_sh, v_st;   // bytes
  int32_t n_pages, H_kv, page;
};

struct WriteParams {
  Pool pool;
  const char* k;
  const char* v;
  int64_t k_st, k_sh, v_st, v_sh;               // bytes
  const int64_t* slots;
  int32_t T, vecs;                              // vectors of a row
};

// write_kernel: a CTA takes kWriteTok tokens; item = (token, K or V, head,
// vector), four independent vectors a thread in flight.  HBM-bound: every
// byte is read once and written once.  65436 tokens of 8 x 128 bf16 (537 MB
// read and written): 92 us, 5.8 TB/s of a plain copy's 6.5; 2 tokens a CTA 113
// us, 4 96 us, 16 92 us; evict-first loads and stores changed nothing beyond
// that.
constexpr int kWriteThreads = 256;
constexpr int kWriteTok = 8;

template <typename V>
__global__ void __launch_bounds__(kWriteThreads) write_kernel(const WriteParams p) {
  __shared__ int64_t s_k[kWriteTok], s_v[kWriteTok];
  const int t0 = (int)blockIdx.x * kWriteTok;
  const int nt = min(kWriteTok, p.T - t0);
  if (threadIdx.x < nt) {
    const int64_t slot = p.slots[t0 + threadIdx.x];
    int64_t ko = -1, vo = -1;
    if (slot >= 0 && slot / p.pool.page < p.pool.n_pages) {
      const int64_t pg = slot / p.pool.page, row = slot % p.pool.page;
      ko = pg * p.pool.k_sp + row * p.pool.k_st;
      vo = pg * p.pool.v_sp + row * p.pool.v_st;
    }
    s_k[threadIdx.x] = ko;
    s_v[threadIdx.x] = vo;
  }
  __syncthreads();
  const int per_kv = p.pool.H_kv * p.vecs, per_tok = 2 * per_kv;
  const int n = nt * per_tok;
  for (int base = threadIdx.x; base < n; base += 4 * kWriteThreads) {
    V x[4];
    char* dst[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + u * kWriteThreads;
      dst[u] = nullptr;
      if (i < n) {
        const int t = i / per_tok, j = i - t * per_tok;
        const bool is_v = j >= per_kv;
        const int jj = is_v ? j - per_kv : j, h = jj / p.vecs, c = jj - h * p.vecs;
        const int64_t off = is_v ? s_v[t] : s_k[t];
        if (off >= 0) {
          const char* src = is_v ? p.v + (int64_t)(t0 + t) * p.v_st + h * p.v_sh
                                 : p.k + (int64_t)(t0 + t) * p.k_st + h * p.k_sh;
          x[u] = *reinterpret_cast<const V*>(src + c * sizeof(V));
          dst[u] = (is_v ? p.pool.v + h * p.pool.v_sh : p.pool.k + h * p.pool.k_sh) + off +
                   c * sizeof(V);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (dst[u]) *reinterpret_cast<V*>(dst[u]) = x[u];
  }
}

struct CommitParams {
  Pool pool;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* ctx;
  const int32_t* path;
  int64_t path_stride;
  const int32_t* path_lens;
  int32_t max_blocks, depth, vecs;
};

// commit_kernel: CTA = (vectors of a request's row, request); a thread owns
// one vector of every row, takes the steps in order and reads eight rows
// before it writes any.  Step i reads node path[i] >= i and writes row i, so
// the row that step j reads (path[j] = i > j) is overwritten by step i only
// after it was read.  Steps that move nothing (path[i] == i) cost no access.
constexpr int kCommitThreads = 128;   // 256: 10.3 us, 64: 10.9 us against 9.9 us (512 requests, 16 steps)
constexpr int kCommitSteps = 128;    // steps staged at a time
constexpr int kCommitRows = 8;       // rows in flight

template <typename V>
__global__ void __launch_bounds__(kCommitThreads) commit_kernel(const CommitParams p) {
  __shared__ int32_t s_sp[kCommitSteps], s_sr[kCommitSteps], s_dp[kCommitSteps],
      s_dr[kCommitSteps];
  const int r = (int)blockIdx.y;
  const int64_t ctx = p.ctx[r];
  const int steps = min(max(p.path_lens[r], 0), p.depth);
  const int u = (int)blockIdx.x * kCommitThreads + threadIdx.x;
  const int per_kv = p.pool.H_kv * p.vecs;
  const bool live = u < 2 * per_kv;
  const bool is_v = u >= per_kv;
  const int uu = is_v ? u - per_kv : u, h = uu / p.vecs, c = uu - h * p.vecs;
  char* base = is_v ? p.pool.v + h * p.pool.v_sh : p.pool.k + h * p.pool.k_sh;
  base += c * sizeof(V);
  const int64_t sp = is_v ? p.pool.v_sp : p.pool.k_sp, st = is_v ? p.pool.v_st : p.pool.k_st;
  const int32_t* tab = p.table + (int64_t)r * p.table_stride;
  for (int i0 = 0; i0 < steps; i0 += kCommitSteps) {
    __syncthreads();
    for (int i = threadIdx.x; i < kCommitSteps; i += kCommitThreads) {
      int32_t a = -1, b = -1, ar = 0, br = 0;
      if (i0 + i < steps && ctx >= 0) {
        const int64_t node = p.path[(int64_t)r * p.path_stride + i0 + i];
        const int64_t src = ctx + node, dst = ctx + i0 + i;
        if (node > i0 + i && src / p.pool.page < p.max_blocks) {
          a = tab[src / p.pool.page];
          b = tab[dst / p.pool.page];
          ar = (int32_t)(src % p.pool.page);
          br = (int32_t)(dst % p.pool.page);
          if ((uint32_t)a >= (uint32_t)p.pool.n_pages || (uint32_t)b >= (uint32_t)p.pool.n_pages)
            a = -1;
        }
      }
      s_sp[i] = a;
      s_sr[i] = ar;
      s_dp[i] = b;
      s_dr[i] = br;
    }
    __syncthreads();
    if (!live) continue;
    const int m = min(kCommitSteps, steps - i0);
    for (int j0 = 0; j0 < m; j0 += kCommitRows) {
      V x[kCommitRows];
#pragma unroll
      for (int j = 0; j < kCommitRows; ++j)
        if (j0 + j < m && s_sp[j0 + j] >= 0)
          x[j] = *reinterpret_cast<const V*>(base + s_sp[j0 + j] * sp + s_sr[j0 + j] * st);
#pragma unroll
      for (int j = 0; j < kCommitRows; ++j)
        if (j0 + j < m && s_sp[j0 + j] >= 0)
          *reinterpret_cast<V*>(base + s_dp[j0 + j] * sp + s_dr[j0 + j] * st) = x[j];
    }
  }
}

// ================================================================ host side
static int elt_bytes(int dtype) {
  return dtype == HALO_DTYPE_F32 ? 4
         : (dtype == HALO_DTYPE_BF16 || dtype == HALO_DTYPE_F16) ? 2 : 0;
}

static int make_pool(const halo_page_pool_t* pool, Pool* out) {
  if (!pool) return fail(HALO_ERR_INVALID_ARG, "page pool is NULL");
  const int e = elt_bytes(pool->dtype);
  if (e == 0) return fail(HALO_ERR_INVALID_ARG, "bad dtype %d", pool->dtype);
  if (pool->n_pages <= 0 || pool->H_kv <= 0 || pool->page_size <= 0 || pool->D <= 0)
    return fail(HALO_ERR_INVALID_ARG, "non-positive pool dimension (n_pages=%d H_kv=%d page_size=%d D=%d)",
                pool->n_pages, pool->H_kv, pool->page_size, pool->D);
  if (!pool->k || !pool->v) return fail(HALO_ERR_INVALID_ARG, "NULL page pool");
  if (((reinterpret_cast<uintptr_t>(pool->k) | reinterpret_cast<uintptr_t>(pool->v)) % e) != 0)
    return fail(HALO_ERR_MISALIGNED, "page pool pointer not aligned to its elements");
  out->k = static_cast<char*>(pool->k);
  out->v = static_cast<char*>(pool->v);
  out->k_sp = pool->k_stride_p * e;
  out->k_sh = pool->k_stride_h * e;
  out->k_st = pool->k_stride_t * e;
  out->v_sp = pool->v_stride_p * e;
  out->v_sh = pool->v_stride_h * e;
  out->v_st = pool->v_stride_t * e;
  out->n_pages = pool->n_pages;
  out->H_kv = pool->H_kv;
  out->page = pool->page_size;
  return HALO_OK;
}

// Every address and stride of the pool, OR-ed: its low bits bound the width
// of a vector access.
static uint64_t pool_bits(const Pool& p) {
  return reinterpret_cast<uint64_t>(p.k) | reinterpret_cast<uint64_t>(p.v) | (uint64_t)p.k_sp |
         (uint64_t)p.k_sh | (uint64_t)p.k_st | (uint64_t)p.v_sp | (uint64_t)p.v_sh |
         (uint64_t)p.v_st;
}

static int vec_bytes(uint64_t bits) {
  return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
}

// Launch of either form; lengths, tables and outputs are checked by the callers.
template <bool STEP>
static int launch_tables(const TablesParams& p, halo_stream_t stream) {
  const size_t smem = (size_t)kTabArrays * p.R * sizeof(int32_t);
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63], [&] {
    e = cudaFuncSetAttribute(tables_kernel<STEP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kTabArrays * kTabMaxReq * (int)sizeof(int32_t));
  });
  if (e != cudaSuccess) return cuda_fail(e, "tables_kernel shared-memory attribute");
  // two tokens a thread before another CTA joins
  const int n_cta = std::min(8, std::max(1, p.T / (2 * kTabThreads)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)n_cta);
  cfg.blockDim = dim3(kTabThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)n_cta;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, tables_kernel<STEP>, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "tables_kernel launch");
  count_launches();
  return HALO_OK;
}

// Sizes that both forms have in common.
static int check_tables(int64_t table_stride, int32_t R, int32_t max_blocks, int32_t free_capacity,
                        int32_t page_size, int32_t max_tokens) {
  if (R < 0 || max_blocks < 0 || free_capacity < 0 || max_tokens < 0 || page_size <= 0)
    return fail(HALO_ERR_INVALID_ARG, "bad size (R=%d max_blocks=%d free=%d max_tokens=%d page_size=%d)",
                R, max_blocks, free_capacity, max_tokens, page_size);
  if (max_tokens > (1 << 30) || free_capacity > (1 << 30))
    return fail(HALO_ERR_UNSUPPORTED, "%d tokens, %d pages", max_tokens, free_capacity);
  if (R > kTabMaxReq) return fail(HALO_ERR_UNSUPPORTED, "%d requests (at most %d)", R, kTabMaxReq);
  if ((int64_t)R * max_blocks > INT_MAX || ((int64_t)max_blocks + 1) * page_size > INT_MAX)
    return fail(HALO_ERR_UNSUPPORTED, "block tables of %d x %d pages of %d are too large", R,
                max_blocks, page_size);
  if (R > 1 && table_stride < max_blocks)
    return fail(HALO_ERR_INVALID_ARG, "block table rows overlap (stride %lld < %d)",
                (long long)table_stride, max_blocks);
  return HALO_OK;
}

static uint32_t magic(int32_t page_size) {
  return (uint32_t)(((1ull << 32) + page_size - 1) / page_size);
}

}  // namespace paged
}  // namespace halo

using namespace halo;

extern "C" int32_t halo_update_block_tables(int32_t* block_tables, int64_t table_stride, int32_t R,
                                            int32_t max_blocks, const int32_t* old_lens,
                                            const int32_t* new_lens, int32_t* free_pages,
                                            int32_t free_capacity, const int32_t* n_free,
                                            int32_t* n_free_out, int32_t page_size,
                                            int32_t max_tokens, int64_t* slots, int64_t* positions,
                                            int32_t* cu_tokens, int32_t* lens,
                                            halo_stream_t stream) {
  using namespace halo::paged;
  const int rc = check_tables(table_stride, R, max_blocks, free_capacity, page_size, max_tokens);
  if (rc != HALO_OK) return rc;
  if ((R > 0 && (!old_lens || !new_lens || !lens || (max_blocks > 0 && !block_tables))) ||
      (free_capacity > 0 && !free_pages) || !n_free || !n_free_out || !cu_tokens ||
      (max_tokens > 0 && (!slots || !positions)))
    return fail(HALO_ERR_INVALID_ARG, "NULL pointer");
  // several CTAs read the lengths, one writes them
  if ((lens < old_lens + R && old_lens < lens + R) || (lens < new_lens + R && new_lens < lens + R))
    return fail(HALO_ERR_INVALID_ARG, "lens overlaps the lengths it is made from");
  return launch_tables<false>(
      TablesParams{block_tables, table_stride, old_lens, new_lens, nullptr, nullptr, nullptr,
                   nullptr, free_pages, n_free, n_free_out, slots, positions, cu_tokens, lens, R, max_blocks,
                   page_size, free_capacity, max_tokens, magic(page_size)}, stream);
}

extern "C" int32_t halo_extend_block_tables(int32_t* block_tables, int64_t table_stride, int32_t R,
                                            int32_t max_blocks, int32_t* held_lens,
                                            const int32_t* context_lens, const int32_t* counts,
                                            int32_t* free_pages, int32_t free_capacity,
                                            int32_t* n_free, int32_t page_size, int32_t max_tokens,
                                            int64_t* slots, int64_t* positions, int32_t* cu_tokens,
                                            int32_t* rows, int32_t* starts,
                                            halo_stream_t stream) {
  using namespace halo::paged;
  const int rc = check_tables(table_stride, R, max_blocks, free_capacity, page_size, max_tokens);
  if (rc != HALO_OK) return rc;
  if ((R > 0 && (!held_lens || !context_lens || !counts || !rows || !starts ||
                 (max_blocks > 0 && !block_tables))) ||
      (free_capacity > 0 && !free_pages) || !n_free || !cu_tokens ||
      (max_tokens > 0 && (!slots || !positions)))
    return fail(HALO_ERR_INVALID_ARG, "NULL pointer");
  // several CTAs read the lengths, one writes rows and starts early and held late
  const auto overlap = [&](const int32_t* a, const int32_t* b) { return a < b + R && b < a + R; };
  if (overlap(rows, held_lens) || overlap(rows, context_lens) || overlap(rows, counts) ||
      overlap(held_lens, context_lens) || overlap(held_lens, counts) ||
      overlap(starts, held_lens) || overlap(starts, context_lens) || overlap(starts, counts) ||
      overlap(starts, rows))
    return fail(HALO_ERR_INVALID_ARG, "held_lens, rows or starts overlap one another or what they "
                "are made from");
  return launch_tables<true>(
      TablesParams{block_tables, table_stride, held_lens, counts, context_lens, rows, starts,
                   held_lens, free_pages, n_free, n_free, slots, positions, cu_tokens, nullptr, R, max_blocks,
                   page_size, free_capacity, max_tokens, magic(page_size)}, stream);
}

extern "C" int32_t halo_write_kv_pages(const halo_page_pool_t* pool, const void* k,
                                       int64_t k_stride_t, int64_t k_stride_h, const void* v,
                                       int64_t v_stride_t, int64_t v_stride_h, int32_t T,
                                       const int64_t* slots, halo_stream_t stream) {
  using namespace halo::paged;
  WriteParams p{};
  int rc = make_pool(pool, &p.pool);
  if (rc != HALO_OK) return rc;
  if (T < 0) return fail(HALO_ERR_INVALID_ARG, "negative token count");
  if (T == 0) return HALO_OK;
  if (!k || !v || !slots) return fail(HALO_ERR_INVALID_ARG, "NULL pointer");
  const int e = elt_bytes(pool->dtype);
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % e)
    return fail(HALO_ERR_MISALIGNED, "k/v pointer not aligned to its elements");
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.k_st = k_stride_t * e;
  p.k_sh = k_stride_h * e;
  p.v_st = v_stride_t * e;
  p.v_sh = v_stride_h * e;
  p.slots = slots;
  p.T = T;
  const int row = pool->D * e;
  const int vb = vec_bytes(pool_bits(p.pool) | reinterpret_cast<uint64_t>(k) |
                           reinterpret_cast<uint64_t>(v) | (uint64_t)p.k_st | (uint64_t)p.k_sh |
                           (uint64_t)p.v_st | (uint64_t)p.v_sh | (uint64_t)row);
  p.vecs = row / vb;
  if ((int64_t)2 * p.vecs * pool->H_kv * kWriteTok > INT_MAX / 2)
    return fail(HALO_ERR_UNSUPPORTED, "a token's rows are too large");
  const unsigned grid = (unsigned)(((int64_t)T + kWriteTok - 1) / kWriteTok);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (vb == 16) write_kernel<uint4><<<grid, kWriteThreads, 0, st>>>(p);
  else if (vb == 8) write_kernel<uint2><<<grid, kWriteThreads, 0, st>>>(p);
  else if (vb == 4) write_kernel<uint32_t><<<grid, kWriteThreads, 0, st>>>(p);
  else write_kernel<uint16_t><<<grid, kWriteThreads, 0, st>>>(p);
  cudaError_t ce = cudaGetLastError();
  if (ce != cudaSuccess) return cuda_fail(ce, "write_kernel launch");
  count_launches();
  return HALO_OK;
}

extern "C" int32_t halo_commit_tree_path(const halo_page_pool_t* pool, const int32_t* block_tables,
                                         int64_t table_stride, int32_t max_blocks, int32_t R,
                                         const int32_t* context_lens, const int32_t* path,
                                         int64_t path_stride, int32_t max_depth,
                                         const int32_t* path_lens, halo_stream_t stream) {
  using namespace halo::paged;
  CommitParams p{};
  int rc = make_pool(pool, &p.pool);
  if (rc != HALO_OK) return rc;
  if (R < 0 || max_depth < 0 || max_blocks < 0)
    return fail(HALO_ERR_INVALID_ARG, "bad size (R=%d max_depth=%d max_blocks=%d)", R, max_depth,
                max_blocks);
  if (R > 65535) return fail(HALO_ERR_UNSUPPORTED, "%d requests (at most 65535)", R);
  if (R == 0 || max_depth == 0 || max_blocks == 0) return HALO_OK;
  if (!block_tables || !context_lens || !path || !path_lens)
    return fail(HALO_ERR_INVALID_ARG, "NULL pointer");
  p.table = block_tables;
  p.table_stride = table_stride;
  p.ctx = context_lens;
  p.path = path;
  p.path_stride = path_stride;
  p.path_lens = path_lens;
  p.max_blocks = max_blocks;
  p.depth = max_depth;
  const int row = pool->D * elt_bytes(pool->dtype);
  const int vb = vec_bytes(pool_bits(p.pool) | (uint64_t)row);
  p.vecs = row / vb;
  const int64_t per = (int64_t)2 * pool->H_kv * p.vecs;
  if (per > INT_MAX / 2) return fail(HALO_ERR_UNSUPPORTED, "a token's rows are too large");
  const dim3 grid((unsigned)((per + kCommitThreads - 1) / kCommitThreads), (unsigned)R);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (vb == 16) commit_kernel<uint4><<<grid, kCommitThreads, 0, st>>>(p);
  else if (vb == 8) commit_kernel<uint2><<<grid, kCommitThreads, 0, st>>>(p);
  else if (vb == 4) commit_kernel<uint32_t><<<grid, kCommitThreads, 0, st>>>(p);
  else commit_kernel<uint16_t><<<grid, kCommitThreads, 0, st>>>(p);
  cudaError_t ce = cudaGetLastError();
  if (ce != cudaSuccess) return cuda_fail(ce, "commit_kernel launch");
  count_launches();
  return HALO_OK;
}
