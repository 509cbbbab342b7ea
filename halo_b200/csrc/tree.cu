// Attention of drafted token trees over the paged K/V cache.
//
// Request r has context_lens[r] cached positions and n_r drafted nodes whose
// K/V rows follow them; node i sees the context and the nodes its mask row
// shows.  For query row (node i, head h) over the positions j it sees
//   s_j = scale q . k_j,  m = max s_j,  l = sum e^{s_j - m},
//   out = sum e^{s_j - m} v_j / l,  lse = m + ln l
// (zeros and -inf where it sees nothing).
#include <climits>
#include <cmath>

#include "halo_common.cuh"

namespace halo {

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);

namespace tree {

struct Params {
  const char* k;
  const char* v;
  int64_t k_sp, k_sh, k_st, v_sp, v_sh, v_st;    // elements
  const char* q;
  int64_t q_st, q_sh;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* ctx;
  const int32_t* cu;
  const uint8_t* mask;
  int64_t mask_stride;
  char* out;
  int64_t out_st, out_sh;
  float* lse;
  float scale_log2;
  int32_t out_f32;
  int32_t R, T, H, G, max_nodes, max_blocks, n_pages, page;
};

// One CTA per query row (node, head), keys dealt to its warps, a lane
// holding D / 32 columns.
constexpr int kWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) tree_rows_kernel(const Params p) {
  constexpr int C = D / 32;
  __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][D];
  const int t = (int)blockIdx.x, h = (int)blockIdx.y, hk = h / p.G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (t >= p.cu[p.R]) return;
  int lo = 0, n = p.R;                 // the request of row t
  while (n > 1) {
    const int half = n >> 1;
    if (p.cu[lo + half] <= t) {
      lo += half;
      n -= half;
    } else {
      n = half;
    }
  }
  const int r = lo, node = t - p.cu[r];
  const int nodes = min(p.cu[r + 1] - p.cu[r], p.max_nodes);
  if (node < 0 || node >= nodes) return;
  const int64_t ctx = max(p.ctx[r], 0);
  const int64_t end = min(ctx + nodes, (int64_t)p.max_blocks * p.page);
  const T* q = reinterpret_cast<const T*>(p.q) + t * p.q_st + h * p.q_sh + lane * C;
  const uint8_t* mask = p.mask + t * p.mask_stride;
  const int32_t* tab = p.table + r * p.table_stride;
  float qf[C], o[C], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    qf[c] = Elem<T>::to_f32(q[c]);
    o[c] = 0.f;
  }
  for (int64_t j = warp; j < end; j += kWarps) {
    if (j >= ctx && !mask[j - ctx]) continue;
    const int32_t pg = tab[j / p.page];
    const int row = (int)(j % p.page);
    const bool in = (uint32_t)pg < (uint32_t)p.n_pages;
    float s = 0.f;
    if (in) {
      const T* k = reinterpret_cast<const T*>(p.k) + pg * p.k_sp + hk * p.k_sh + row * p.k_st + lane * C;
#pragma unroll
      for (int c = 0; c < C; ++c) s = fmaf(qf[c], Elem<T>::to_f32(k[c]), s);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= p.scale_log2;
    const float mn = fmaxf(m, s);
    const float a = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float w = s == -INFINITY ? 0.f : exp2f(s - mn);
    l = l * a + w;
    const T* v = reinterpret_cast<const T*>(p.v) + (in ? pg * p.v_sp + hk * p.v_sh + row * p.v_st + lane * C : 0);
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = o[c] * a + (in ? w * Elem<T>::to_f32(v[c]) : 0.f);
    m = mn;
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int c = 0; c < C; ++c) s_o[warp][lane * C + c] = o[c];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w]);
  const int d = threadIdx.x;
  float acc = 0.f;
  for (int w = 0; w < kWarps; ++w) {
    const float e = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - M);
    L = fmaf(s_l[w], e, L);
    if (d < D) acc = fmaf(s_o[w][d], e, acc);
  }
  if (d < D) {
    const float x = L > 0.f ? acc / L : (L == L ? 0.f : L);
    const int64_t at = t * p.out_st + h * p.out_sh + d;
    if (p.out_f32) reinterpret_cast<float*>(p.out)[at] = x;
    else reinterpret_cast<T*>(p.out)[at] = Elem<T>::from_f32(x);
  }
  if (d == 0 && p.lse)
    p.lse[(int64_t)t * p.H + h] = L > 0.f ? (M + log2f(L)) * kLn2 : (L == L ? -INFINITY : L);
}

}  // namespace tree

// ================================================================ host side
static bool rows16(const void* p, int64_t a, int64_t b, int64_t c, int elt) {
  return ((reinterpret_cast<uintptr_t>(p) | (uint64_t)(a * elt) | (uint64_t)(b * elt) |
           (uint64_t)(c * elt)) & 15) == 0;
}

static int tree_check(const halo_page_pool_t* pool, const halo_tree_problem_t* pb) {
  if (!pool || !pb) return fail(HALO_ERR_INVALID_ARG, "page pool/problem is NULL");
  if (pool->dtype != HALO_DTYPE_BF16 && pool->dtype != HALO_DTYPE_F16)
    return fail(HALO_ERR_UNSUPPORTED, "tree attention needs bf16 or fp16 (dtype %d)", pool->dtype);
  if (pool->D != 64 && pool->D != 128)
    return fail(HALO_ERR_UNSUPPORTED, "tree attention head_dim %d (64 or 128)", pool->D);
  if (pool->n_pages <= 0 || pool->H_kv <= 0 || pool->page_size <= 0)
    return fail(HALO_ERR_INVALID_ARG, "non-positive pool dimension (n_pages=%d H_kv=%d page_size=%d)",
                pool->n_pages, pool->H_kv, pool->page_size);
  if (pool->page_size % 8)
    return fail(HALO_ERR_UNSUPPORTED, "page_size %d is not a multiple of 8", pool->page_size);
  if (pb->R < 0 || pb->T < 0 || pb->H <= 0 || pb->max_nodes < 0 || pb->max_blocks < 0)
    return fail(HALO_ERR_INVALID_ARG, "bad size (R=%d T=%d H=%d max_nodes=%d max_blocks=%d)", pb->R,
                pb->T, pb->H, pb->max_nodes, pb->max_blocks);
  if (pb->H % pool->H_kv)
    return fail(HALO_ERR_INVALID_ARG, "H=%d not divisible by H_kv=%d", pb->H, pool->H_kv);
  if (pb->max_nodes > 1024)
    return fail(HALO_ERR_UNSUPPORTED, "%d nodes a request (at most 1024)", pb->max_nodes);
  if ((int64_t)pb->max_blocks * pool->page_size + 1024 > INT_MAX)
    return fail(HALO_ERR_UNSUPPORTED, "block tables of %d pages of %d are too long", pb->max_blocks,
                pool->page_size);
  if (!(pb->scale > 0.f) || !std::isfinite(pb->scale))
    return fail(HALO_ERR_UNSUPPORTED, "tree attention needs a positive finite scale");
  return HALO_OK;
}

}  // namespace halo

using namespace halo;

extern "C" int64_t halo_tree_workspace_bytes(const halo_page_pool_t* pool,
                                             const halo_tree_problem_t* pb) {
  const int rc = tree_check(pool, pb);
  return rc != HALO_OK ? rc : 0;
}

extern "C" int32_t halo_tree_attention(const halo_page_pool_t* pool, const halo_tree_problem_t* pb,
                                       void* workspace, int64_t workspace_bytes,
                                       halo_stream_t stream) {
  int rc = tree_check(pool, pb);
  if (rc != HALO_OK) return rc;
  (void)workspace;
  (void)workspace_bytes;
  if (pb->R == 0 || pb->T == 0 || pb->max_nodes == 0) return HALO_OK;
  if (!pool->k || !pool->v || !pb->q || !pb->out || !pb->context_lens || !pb->cu_nodes ||
      !pb->mask || (pb->max_blocks > 0 && !pb->block_tables))
    return fail(HALO_ERR_INVALID_ARG, "NULL pointer");
  if (pb->out_dtype != HALO_DTYPE_F32 && pb->out_dtype != pool->dtype)
    return fail(HALO_ERR_UNSUPPORTED, "out dtype must be fp32 or the pool's dtype");
  if (!rows16(pool->k, pool->k_stride_p, pool->k_stride_h, pool->k_stride_t, 2) ||
      !rows16(pool->v, pool->v_stride_p, pool->v_stride_h, pool->v_stride_t, 2) ||
      pool->k_stride_t <= 0 || pool->v_stride_t <= 0)
    return fail(HALO_ERR_MISALIGNED, "page rows must be 16-byte aligned");
  if (!rows16(pb->q, pb->q_stride_t, pb->q_stride_h, 0, 2))
    return fail(HALO_ERR_MISALIGNED, "q rows must be 16-byte aligned");
  if (!rows16(pb->out, pb->out_stride_t, pb->out_stride_h, 0,
              pb->out_dtype == HALO_DTYPE_F32 ? 4 : 2))
    return fail(HALO_ERR_MISALIGNED, "out rows must be 16-byte aligned");
  if (pb->H > 65535) return fail(HALO_ERR_UNSUPPORTED, "%d heads", pb->H);
  tree::Params p{};
  p.k = static_cast<const char*>(pool->k);
  p.v = static_cast<const char*>(pool->v);
  p.k_sp = pool->k_stride_p;
  p.k_sh = pool->k_stride_h;
  p.k_st = pool->k_stride_t;
  p.v_sp = pool->v_stride_p;
  p.v_sh = pool->v_stride_h;
  p.v_st = pool->v_stride_t;
  p.q = static_cast<const char*>(pb->q);
  p.q_st = pb->q_stride_t;
  p.q_sh = pb->q_stride_h;
  p.table = pb->block_tables;
  p.table_stride = pb->table_stride;
  p.ctx = pb->context_lens;
  p.cu = pb->cu_nodes;
  p.mask = pb->mask;
  p.mask_stride = pb->mask_stride;
  p.out = static_cast<char*>(pb->out);
  p.out_st = pb->out_stride_t;
  p.out_sh = pb->out_stride_h;
  p.lse = pb->lse;
  p.scale_log2 = pb->scale * kLog2e;
  p.out_f32 = pb->out_dtype == HALO_DTYPE_F32;
  p.R = pb->R;
  p.T = pb->T;
  p.H = pb->H;
  p.G = pb->H / pool->H_kv;
  p.max_nodes = pb->max_nodes;
  p.max_blocks = pb->max_blocks;
  p.n_pages = pool->n_pages;
  p.page = pool->page_size;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)pb->T, (unsigned)pb->H);
  const int threads = tree::kWarps * 32;
  if (pool->dtype == HALO_DTYPE_BF16) {
    if (pool->D == 128) tree::tree_rows_kernel<__nv_bfloat16, 128><<<grid, threads, 0, st>>>(p);
    else tree::tree_rows_kernel<__nv_bfloat16, 64><<<grid, threads, 0, st>>>(p);
  } else {
    if (pool->D == 128) tree::tree_rows_kernel<__half, 128><<<grid, threads, 0, st>>>(p);
    else tree::tree_rows_kernel<__half, 64><<<grid, threads, 0, st>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "tree_rows_kernel launch");
  count_launches();
  return HALO_OK;
}
