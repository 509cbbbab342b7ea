// Attention of drafted token trees over the paged K/V cache.
//
// Request r has context_lens[r] cached positions and n_r drafted nodes whose
// K/V rows follow them; node i sees the context and the nodes its mask row
// shows.  For query row (node i, head h) over the positions j it sees
//   s_j = scale q . k_j,  m = max s_j,  l = sum e^{s_j - m},
//   out = sum e^{s_j - m} v_j / l,  lse = m + ln l
// (zeros and -inf where it sees nothing).
//
// The n_r * G query rows that share a K/V head (G = H / H_kv) go through the
// tensor cores together, so a K/V row is read once for all of them (once for
// each 256 of them).  Up to about 64 rows the cache's bytes bound the kernel;
// at 256 rows bytes, products and exponentials come out about level.
//
// Split: a unit is 128 positions of one (request, K/V head, row group), and
// the units of all requests, in that order, are cut into one equal run per
// SM.  The lengths are read on the device, so the cut is even for any mix of
// them and nothing depends on the host knowing one.  A (request, head, group)
// that lies in one run is finished there; the parts of others go to the
// workspace as (m, l, o) and tree_merge_kernel joins them.
#include <algorithm>
#include <climits>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "halo_common.cuh"
#include "running_max.cuh"
#include "umma.cuh"

namespace halo {

int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);
int device_sms();

namespace tree {

constexpr int kBN = 128;               // positions of a tile (a unit)
constexpr int kThreads = 640;          // tree_kernel
constexpr uint32_t kTmemCols = 512;
constexpr int kBadSlots = 8;

struct alignas(64) Params {
  CUtensorMap kmap;                    // see encode_pool
  CUtensorMap vmap;
  const char* q;
  int64_t q_st, q_sh;                  // elements
  const char* v;
  int64_t v_sp, v_sh, v_st;            // elements
  const int32_t* table;
  int64_t table_stride;
  const int32_t* ctx;
  const int32_t* cu;
  const int32_t* starts;               // where a request's rows begin: cu itself unless given
  const uint8_t* mask;
  int64_t mask_stride;
  char* out;
  int64_t out_st, out_sh;
  float* lse;                          // never null: in the workspace if not asked for
  float scale_log2;                    // softmax scale * log2(e)
  float headroom;                      // of the running maximum, in raw scores
  int32_t out_f32;
  int32_t R, T, H, H_kv, G, max_nodes, max_blocks, n_pages, page, box;
  struct Desc* desc;                   // workspace: one a CTA
  float* part;                         // workspace: two slots a CTA
  unsigned int* err;
};

// What the merge has to know of the segment that holds a CTA's first unit.
struct alignas(64) Desc {
  int64_t start;                       // units before the segment's first tile
  int64_t quot;                        // all units: quot * CTAs + rem
  int32_t rem;
  int32_t nt;                          // the segment's tiles
  int32_t cu0, hk, row0, rows;         // row0: the group's first row of the request
};

// A part of a cut segment in the workspace: o [RG][D], then (m of the raw
// scores, l) [RG][2], fp32.
template <int D>
__host__ __device__ constexpr int64_t part_floats(int RG) {
  return (int64_t)RG * (D + 2);
}

// A K/V tile in shared memory: 128 rows of D / 64 column blocks of 128 bytes,
// swizzled.  A block is contiguous, or (PAIR) each 8 rows of both blocks are:
// a copy cannot cross a page, so a tile of pages whose rows are an odd multiple
// of 8 would take 32 copies of 8 rows and one block.
template <int D, bool PAIR>
struct Tile {
  static_assert(!PAIR || D == 128, "pairs of column blocks");
  static constexpr bool kPair = PAIR;
  static constexpr int kBlocks = D / 64;
  static constexpr int kBlockBytes = kBN * 128;
  static constexpr int kGroup = PAIR ? 2048 : 1024;       // from 8 rows to the next 8
  static constexpr int kNextBlock = PAIR ? 1024 : kBlockBytes;
};

// tree_kernel: QT query tiles of 128 rows.
template <int D, int QT, bool PAIR>
struct Geom : Tile<D, PAIR> {
  using Tile<D, PAIR>::kBlocks;
  using Tile<D, PAIR>::kBlockBytes;
  static constexpr int kTileBytes = kBlocks * kBlockBytes;
  // as many K and V tiles in flight as 227 KB hold beside QT query tiles
  static constexpr int kStK = D == 64 ? 6 : 3;
  static constexpr int kStV = D == 64 ? 6 : (QT == 1 ? 3 : 2);
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = QT * kTileBytes;
  static constexpr int kOffV = kOffK + kStK * kTileBytes;
  static constexpr int kOffMl = kOffV + kStV * kTileBytes;   // maxima [2][2][128]
  static constexpr int kOffBar = kOffMl + 2048;
  static constexpr int kSmemBytes = kOffBar + 1024;
  static constexpr uint32_t kColO = 256;
};

// tree_few_kernel: NR (16, 32 or 64) query rows.
template <int D, int NR, bool PAIR>
struct FewGeom : Tile<D, PAIR> {
  using Tile<D, PAIR>::kBlocks;
  using Tile<D, PAIR>::kBlockBytes;
  // Softmax groups of four warps.  Four where 64 rows' softmax is longer than a
  // tile's bytes (64 columns): 64 requests of 16 nodes on 1200 positions 75 us
  // and 84 with two, 8 on 32768 positions 154 to 160 and 173, but 23.2 and 20.8
  // on 40 positions.  At 128 columns two: 202 and 204 us on 32768 positions, 54
  // (four) and 51.5 on 300.  32 rows in four groups of 8 leave no registers for
  // V's producer: 111 and 120 us on pages of 64, 226 and 148 on pages of 8.
  static constexpr int kGroups = D == 64 && NR == 64 ? 4 : 2;
  static constexpr int kSoft = kGroups * 128;                  // their threads
  // a warp more for V's copies where the registers of 64 rows leave room
  static constexpr int kThreads = 128 + kSoft + (NR == 64 ? 0 : 32);
  static constexpr int kTileBytes = kBlocks * kBlockBytes;
  static constexpr int kQBytes = NR * D * 2;
  static constexpr int kPBytes = (NR == 64 ? 2 : 1) * kBlockBytes;
  // two buffers of P where a tile's bytes take less than P V and its waits
  static constexpr int kPBuf = D == 64 ? 2 : 1;
  static constexpr int kStK = D == 64 ? (NR == 64 ? 4 : 5) : 3;
  static constexpr int kStV = D == 64 ? (NR == 64 ? 4 : 5) : (NR == 64 ? 2 : 3);
  static constexpr int kOffK = 0;
  static constexpr int kOffV = kStK * kTileBytes;
  static constexpr int kOffP = kOffV + kStV * kTileBytes;
  static constexpr int kOffQ = kOffP + kPBuf * kPBytes;        // two buffers
  static constexpr int kOffRed = kOffQ + 2 * kQBytes;          // see FewShared
  static constexpr int kOffBar = kOffRed + 2048;
  static constexpr int kSmemBytes = kOffBar + 1024;
  static constexpr uint32_t kColO = 2 * NR;                    // S 2 x NR, O 2 NR
};
static_assert(FewGeom<128, 64, true>::kSmemBytes <= 232448 &&
              FewGeom<128, 32, true>::kSmemBytes <= 232448 &&
              FewGeom<64, 64, false>::kSmemBytes <= 232448 &&
              FewGeom<64, 32, false>::kSmemBytes <= 232448 &&
              Geom<128, 1, true>::kSmemBytes <= 232448 && Geom<128, 2, true>::kSmemBytes <= 232448 &&
              Geom<64, 2, false>::kSmemBytes <= 232448, "227 KB of shared memory");

struct FewShared {
  float red[4][64];                    // per warp and row
  float m[64], fac[64];                // running maximum; its latest rescale, or 1 / l
  int64_t off[64];                     // output element of each row
};
static_assert(sizeof(FewShared) <= 2048, "scratch of tree_few_kernel");


// ---- the units of a request
struct Req {
  int ctx, end, nodes, cu0, nt, ng;
};

struct Bars {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[6], k_empty[6], v_full[6], v_ready[6], v_empty[6];
  uint64_t s_full[2], s_free[2], p_full[4], pv_done[2], mma_done[2], turn[2];
  int64_t scan[20];
  int64_t base0, u0, u1;
  uint32_t tmem_base;
  int abort_flag, r0, odd;             // odd: an output element is not finite
  Req req0;
  int bad[kBadSlots];
};
static_assert(sizeof(Bars) <= 1024, "barrier block");

// Bounded wait that also ends when another role gave up.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, Bars* bs,
                                         unsigned int* err) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    for (int i = 0; i < 8; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(&bs->abort_flag)) return false;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      set_device_error(err, static_cast<unsigned int>(-HALO_ERR_TIMEOUT));
      *reinterpret_cast<volatile int*>(&bs->abort_flag) = 1;
      return false;
    }
  }
}

// Units that a segment weighs beside its tiles: query rows, first maxima,
// epilogue (about 5 us, against 1.6 us a tile of few rows and 3 us of many).
// They come before its tiles, so a cut among them cuts nothing.  44 trees of
// 34 to 94 nodes on 156 positions: 78 us with 1, 65 us with 3 or 4; 32 decode
// requests of 17 to 16000 positions: 166 us with 1, 157 us with 2 or 3.
template <int RG>
constexpr int kSetup = RG <= 64 ? 3 : 4;

template <int RG>
__device__ __forceinline__ Req load_req(const Params& p, int r) {
  Req q;
  const int lim = p.max_blocks * p.page;
  q.cu0 = min(max(p.starts[r], 0), p.T);
  q.nodes = min(min(max(p.cu[r + 1] - max(p.cu[r], 0), 0), p.max_nodes), p.T - q.cu0);
  q.ctx = min(max(p.ctx[r], 0), lim);
  q.end = min(q.ctx + q.nodes, lim);
  q.ng = (q.nodes * p.G + RG - 1) / RG;
  q.nt = q.nodes > 0 ? max(1, (q.end + kBN - 1) / kBN) : 0;
  return q;
}
template <int RG>
__device__ __forceinline__ int64_t units_of(const Req& q, int H_kv) {
  return (int64_t)(q.nt + kSetup<RG>) * (q.ng * H_kv);
}

// One (request, head, group) part of a CTA's run: tiles [t0, t1) of nt.
struct Seg {
  int hk, row0, rows, t0, t1;
  bool whole, first;
};

// Walks a CTA's run segment by segment; every role keeps its own.
template <int RG>
struct Walk {
  int64_t u, u1, base, units;
  int r;
  bool begun;
  Req q;
  __device__ __forceinline__ Walk(const Params& p, int r0, const Req& q0, int64_t base0, int64_t a,
                                  int64_t b)
      : u(a), u1(b), base(base0), r(r0), begun(false), q(q0) {
    units = units_of<RG>(q, p.H_kv);
  }
  __device__ __forceinline__ bool next(const Params& p, Seg& s) {
    constexpr int W = kSetup<RG>;
    while (u < u1) {
      while (u - base >= units) {
        base += units;
        q = load_req<RG>(p, ++r);
        units = units_of<RG>(q, p.H_kv);
      }
      const int64_t local = u - base;
      const int len = q.nt + W;
      // 32-bit division where it serves
      const int hg = (local >> 31) == 0 ? (int)((uint32_t)local / (uint32_t)len)
                                        : (int)(local / len);
      const int a = (int)(local - (int64_t)hg * len);
      const int b = (int)min((int64_t)len, a + (u1 - u));
      u += b - a;
      s.t0 = max(a - W, 0);
      s.t1 = b - W;
      if (s.t1 <= s.t0) continue;          // set-up units alone
      s.hk = hg / q.ng;
      s.row0 = (hg - s.hk * q.ng) * RG;
      s.rows = min(RG, q.nodes * p.G - s.row0);
      s.whole = s.t0 == 0 && s.t1 == q.nt;
      s.first = !begun;
      begun = true;
      return true;
    }
    return false;
  }
};

// ---- TMEM loads of 8 / 16 columns (the 32-column form is in umma.cuh)
__device__ __forceinline__ void tmem_ld(uint32_t a, float (&v)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                 "=r"(r[6]), "=r"(r[7])
               : "r"(a));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld(uint32_t a, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(a));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld(uint32_t a, float (&v)[32]) { umma::tmem_ld32(a, v); }

__device__ __forceinline__ void tmem_st(uint32_t a, const float (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a),
               "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
               "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
               "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7]))
               : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t a, const float (&v)[16]) {
  umma::tmem_st16u(a, reinterpret_cast<const uint32_t*>(v));
}
__device__ __forceinline__ void tmem_st(uint32_t a, const float (&v)[32]) { umma::tmem_st32(a, v); }

// ---- packed fp32 pairs, three-way maximum
__device__ __forceinline__ uint64_t f2pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2unpack(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Weights are 2^kLift e^{scale (s - m)}.  fp16 has steps of 2^-24 below 2^-14,
// so small weights would be lost from P V while the row sum counts them: lifted
// by 7 they reach 2^15 beside a headroom of 2^8 (fp16 ends at 2^16) and are off
// by 2^-32 of the largest at most.  bf16 has fp32's exponents.  The factor is in
// l and o alike; only the log-sum-exp takes it out.
template <typename T>
constexpr float kLift = Elem<T>::kDtype == HALO_DTYPE_F16 ? 7.f : 0.f;

// Weights of a pair of raw scores: their 16-bit values (hi) and remainders
// (lo); the fp32 pair is returned for the row sum.
template <typename T>
__device__ __forceinline__ uint64_t weigh(float s0, float s1, uint64_t sc2, uint64_t nm2,
                                          uint32_t& hi, uint32_t& lo) {
  float x0, x1, h0, h1;
  f2unpack(ffma2(fadd2(f2pack(s0, s1), nm2), sc2, f2pack(kLift<T>, kLift<T>)), x0, x1);
  const float a = ex2(x0), b = ex2(x1);
  if constexpr (Elem<T>::kDtype == HALO_DTYPE_BF16) {   // truncated: one byte permute a pair
    hi = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    h0 = __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
    h1 = __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
  } else {
    hi = Elem<T>::pack(a, b);
    Elem<T>::unpack(hi, h0, h1);
  }
  const uint64_t p2 = f2pack(a, b);
  float r0, r1;
  f2unpack(ffma2(f2pack(h0, h1), f2pack(-1.f, -1.f), p2), r0, r1);
  lo = Elem<T>::pack(r0, r1);
  return p2;
}

__device__ __forceinline__ void tmem_st8u(uint32_t a, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]),
               "r"(v[7])
               : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// Asynchronous 16-byte copy to shared memory; zeros where `in` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(in ? 16 : 0)
               : "memory");
}

__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int c0, int c1,
                                            int c2, int c3, int c4, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
      ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2),
        "r"(c3), "r"(c4), "r"(smem_addr(bar))
      : "memory");
}

// A value the compiler cannot see through: keeps it from holding every
// unrolled MMA's descriptor in a register across the loop.
__device__ __forceinline__ uint64_t opaque(uint64_t v) {
  asm volatile("mov.b64 %0, %0;" : "+l"(v));
  return v;
}

template <typename T>
__device__ __forceinline__ bool bad16(uint32_t x) {   // inf or NaN in the low 16 bits
  constexpr uint32_t e = Elem<T>::kDtype == HALO_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
  return (x & e) == e;
}

// ln of sum e^{scale s} from the maximum of the raw scores and the sum of weights.
template <typename T>
__device__ __forceinline__ float log_sum(float m, float l, float scale_log2) {
  return l > 0.f ? fmaf(m, scale_log2, log2f(l) - kLift<T>) * kLn2 : (l == l ? -INFINITY : l);
}

// Weight of a state in a join.  Where it would end as 0 it stays the smallest
// normal number, which is as near to it: an infinity of the state stays one.
__device__ __forceinline__ float join_weight(float m, float top, float scale_log2) {
  return fmaxf(ex2(excess(m, top) * scale_log2), 1.17549435e-38f);
}

// Barrier `id` of N softmax threads that tells whether any of them voted.
template <int N>
__device__ __forceinline__ bool vote_bar(int id, bool vote) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(vote ? 1u : 0u), "r"(id), "n"(N)
      : "memory");
  return any != 0;
}

// ---- parts of both kernels

// The CTA's run [c U / C, (c + 1) U / C) of the U units of all requests, and
// the request (bs->r0, beginning at unit bs->base0) that holds its first.
// Ends without a barrier: bs->r0 holds after the caller's next one.
template <int RG, int NT>
__device__ __forceinline__ void find_run(const Params& p, Bars* bs, int64_t& u0, int64_t& u1,
                                         int64_t& U) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto prefix = [&](int64_t v, int64_t& total) {   // inclusive, over the CTA
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) bs->scan[warp] = v;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      if (w < warp) v += bs->scan[w];
      total += bs->scan[w];
    }
    return v;
  };
  Req q;
  auto units = [&](int r) -> int64_t {
    if (r >= p.R) return 0;
    q = load_req<RG>(p, r);
    return units_of<RG>(q, p.H_kv);
  };
  int64_t mine = 0, incl = 0;
  U = 0;
  for (int r0 = 0; r0 < p.R; r0 += NT) {
    int64_t t;
    mine = units(r0 + threadIdx.x);
    incl = prefix(mine, t);
    U += t;
  }
  if ((U >> 20) == 0) {                // 32-bit divisions (a grid has < 2^12 CTAs)
    u0 = (uint32_t)(blockIdx.x * (uint32_t)U) / gridDim.x;
    u1 = (uint32_t)((blockIdx.x + 1) * (uint32_t)U) / gridDim.x;
  } else {
    u0 = (int64_t)blockIdx.x * U / gridDim.x;
    u1 = (int64_t)(blockIdx.x + 1) * U / gridDim.x;
  }
  if (threadIdx.x == 0) {              // for restore, which comes last
    bs->u0 = u0;
    bs->u1 = u1;
  }
  {
    int64_t before = 0;
    for (int r0 = 0; r0 < p.R; r0 += NT) {
      int64_t t = U;
      if (p.R > NT) {                // else the scan above holds
        mine = units(r0 + threadIdx.x);
        incl = prefix(mine, t);
      }
      const int64_t lo = before + incl - mine;
      if (mine > 0 && lo <= u0 && u0 < lo + mine) {
        bs->r0 = r0 + threadIdx.x;
        bs->req0 = q;
        bs->base0 = lo;
      }
      before += t;
    }
  }
}

// One thread: the segment that holds the run's first unit, for the merge.
template <int RG>
__device__ __forceinline__ void write_desc(const Params& p, const Bars* bs, int64_t u0, int64_t U) {
  Desc d{};
  d.quot = U / gridDim.x;
  d.rem = (int32_t)(U - d.quot * gridDim.x);
  if (u0 < U) {
    const Req& q = bs->req0;
    const int len = q.nt + kSetup<RG>;
    const int hg = (int)((u0 - bs->base0) / len);
    d.start = bs->base0 + (int64_t)hg * len + kSetup<RG>;
    d.nt = q.nt;
    d.cu0 = q.cu0;
    d.hk = hg / q.ng;
    d.row0 = (hg - d.hk * q.ng) * RG;
    d.rows = min(RG, q.nodes * p.G - d.row0);
  }
  p.desc[blockIdx.x] = d;
}

// Producer warp: the run's tiles through a ring, K's (KIND 1), V's (KIND 2)
// or both (KIND 3).  A warp for each where tiles are short: issuing one takes
// 500 to 1000 clocks (8 boxes of 16 rows), as long as its bytes at 64 columns.
// SKIP: in segments of at most 128 rows only one of the two streams reads a
// tile.
template <int RG, class Gm, bool SKIP, int KIND>
__device__ __forceinline__ void produce(const Params& p, Bars* bs, unsigned char* smem,
                                        Walk<RG>& walk) {
  constexpr int SK = Gm::kStK, SV = Gm::kStV;
  const int lane = threadIdx.x & 31;
  Seg s{};
  const int n_box = kBN / p.box, n_iss = Gm::kPair ? n_box : n_box * Gm::kBlocks;   // at most 16
  const int blk = lane / n_box, bx = lane - blk * n_box;
  const uint32_t dst = blk * Gm::kBlockBytes + bx * (p.box >> 3) * Gm::kGroup;
  const int step_page = kBN / p.page, step_row = kBN - step_page * p.page;
  int nk = 0, nv = 0;             // K and V tiles issued
  bool ok = true;
  // one tile's boxes into a ring stage, after its previous use
  auto issue = [&](int n, int st, uint64_t* full, uint64_t* empty, int off, const CUtensorMap* map,
                   int row, int page, uint32_t absent) {
    const int i = n % st;
    if (n >= st) ok = __all_sync(0xffffffffu, wait_bar(&empty[i], (n / st - 1) & 1, bs, p.err));
    if (!ok) return;
    if (lane == 0) {
      mbar_arrive_expect_tx(&full[i], Gm::kTileBytes);
      if (absent) mbar_arrive_n(&empty[i], absent);
    }
    __syncwarp();
    if (lane < n_iss) {
      unsigned char* to = smem + off + i * Gm::kTileBytes + dst;
      if constexpr (Gm::kPair) tma_load_5d(to, map, 0, row, 0, s.hk, page, &full[i]);
      else tma_load_4d(to, map, blk * 64, row, s.hk, page, &full[i]);
    }
  };
  while (ok && walk.next(p, s)) {
    const int32_t* tab = p.table + (int64_t)walk.r * p.table_stride;
    const uint32_t absent = SKIP && s.rows <= 128 ? 1u : 0u;   // streams that skip a tile
    // this lane's box: position, table entry and row in the page
    int pos = s.t0 * kBN + bx * p.box;
    int idx = pos / p.page, row = pos - idx * p.page;
    auto entry = [&]() { return lane < n_iss && pos < walk.q.end ? tab[idx] : -1; };
    int pg = entry();
    for (int t = s.t0; t < s.t1 && ok; ++t) {
      const int page = (uint32_t)pg < (uint32_t)p.n_pages ? pg : p.n_pages;   // outside: zeros
      const int this_row = row;
      pos += kBN;
      idx += step_page;
      row += step_row;
      if (row >= p.page) {
        row -= p.page;
        ++idx;
      }
      if (t + 1 < s.t1) pg = entry();      // the next tile's page, ahead of the waits
      if (KIND & 1) {
        issue(nk, SK, bs->k_full, bs->k_empty, Gm::kOffK, &p.kmap, this_row, page, absent);
        if (!ok) break;
        ++nk;
      }
      if (KIND & 2) {
        issue(nv, SV, bs->v_full, bs->v_empty, Gm::kOffV, &p.vmap, this_row, page, absent);
        if (!ok) break;
        ++nv;
      }
    }
  }
  // every copy issued lands before the CTA can exit
  if (lane == 0) {
    for (int i = 0; i < SK; ++i) {
      const int n = (nk - i + SK - 1) / SK;
      if (n > 0) mbar_wait(&bs->k_full[i], (n - 1) & 1, p.err);
    }
    for (int i = 0; i < SV; ++i) {
      const int n = (nv - i + SV - 1) / SV;
      if (n > 0) mbar_wait(&bs->v_full[i], (n - 1) & 1, p.err);
    }
  }
}

// Cleaner warp: passes every V tile on, cleaned where it reaches behind the
// context: rows behind the last node and elements that are not finite become
// zero (a weight of zero would turn them into NaN).  bs->bad[segment] tells
// whether a node's element was taken out; bad_sum gives it back.
// `begin` runs at the start of every segment.
template <typename T, int D, int RG, class Gm, class F>
__device__ __forceinline__ void clean(const Params& p, Bars* bs, unsigned char* smem,
                                      Walk<RG>& walk, F begin) {
  constexpr int SV = Gm::kStV;
  const int lane = threadIdx.x & 31;
  Seg s;
  int g = 0, si = 0;
  bool ok = true;
  volatile int* bad = &bs->bad[0];
  while (ok && walk.next(p, s)) {
    if (lane == 0) bad[si % kBadSlots] = 0;
    __syncwarp();
    ok = begin();
    if (!ok) break;
    for (int t = s.t0; t < s.t1; ++t, ++g) {
      const int iv = g % SV;
      ok = __all_sync(0xffffffffu, wait_bar(&bs->v_full[iv], (g / SV) & 1, bs, p.err));
      if (!ok) break;
      const int lo = max(0, walk.q.ctx - t * kBN), end = walk.q.end - t * kBN;
      if (lo < kBN) {
        bool any = false;
        const int n = (kBN - lo) * (D / 8);
        for (int i = lane; i < n; i += 32) {
          const int row = lo + i / (D / 8), c = i % (D / 8);
          uint4* w = reinterpret_cast<uint4*>(smem + Gm::kOffV + iv * Gm::kTileBytes +
                                              (c >> 3) * Gm::kNextBlock + (row >> 3) * Gm::kGroup +
                                              (row & 7) * 128 + (((c & 7) ^ (row & 7)) << 4));
          if (row >= end) {
            *w = make_uint4(0, 0, 0, 0);
            continue;
          }
          uint4 x = *w;
          uint32_t e[4] = {x.x, x.y, x.z, x.w};
          bool hit = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (bad16<T>(e[k])) {
              e[k] &= 0xFFFF0000u;
              hit = true;
            }
            if (bad16<T>(e[k] >> 16)) {
              e[k] &= 0xFFFFu;
              hit = true;
            }
          }
          if (hit) {
            *w = make_uint4(e[0], e[1], e[2], e[3]);
            any = true;
          }
        }
        if (any) bad[si % kBadSlots] = 1;
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bs->v_ready[iv]);
    }
    ++si;
  }
}

// Sum of the non-finite V elements, in column `col`, of the nodes at positions
// [a, b) that query row t sees: its weights are positive, so each adds itself
// to the row's output.
template <typename T>
__device__ __noinline__ float bad_sum(const Params& p, int r, int t, int ctx, int a, int b, int hk,
                                      int col) {
  float o = 0.f;
  for (int pos = a; pos < b; ++pos) {
    if (!p.mask[(int64_t)t * p.mask_stride + pos - ctx]) continue;
    const int pg = p.table[(int64_t)r * p.table_stride + pos / p.page];
    if ((uint32_t)pg >= (uint32_t)p.n_pages) continue;
    const float y = Elem<T>::to_f32(reinterpret_cast<const T*>(
        p.v)[pg * p.v_sp + hk * p.v_sh + (pos % p.page) * p.v_st + col]);
    if (!isfinite(y)) o += y;
  }
  return o;
}

// ---- infinities of the context.  The context is not cleaned, so an infinity of
// it times a remainder of zero, or of the other sign, makes the output element
// NaN, where the definition gives the infinity.  Such elements are formed again
// when the CTA's run is done: calls in the epilogues cost up to 27 % (16 rows of 64
// columns 97 -> 123 us), calls in the merge 0.7 us of every call.

// Warp: sum of the V elements that are not finite, in column `col`, of the
// positions in [a, b) that query row t sees.
template <typename T>
__device__ __noinline__ float seen_sum(const Params& p, int r, int t, int ctx, int a, int b, int hk,
                                       int col) {
  const T* v = reinterpret_cast<const T*>(p.v) + hk * p.v_sh + col;
  const uint8_t* mask = p.mask + (int64_t)t * p.mask_stride;
  float o = 0.f;
#pragma unroll 1
  for (int pos = a + (int)(threadIdx.x & 31); pos < b; pos += 32) {
    const int idx = pos / p.page, row = pos - idx * p.page;
    const int pg = p.table[(int64_t)r * p.table_stride + idx];
    if ((uint32_t)pg >= (uint32_t)p.n_pages || (pos >= ctx && !mask[pos - ctx])) continue;
    const float y = Elem<T>::to_f32(v[pg * p.v_sp + row * p.v_st]);
    if (!isfinite(y)) o += y;
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) o += __shfl_xor_sync(0xffffffffu, o, d);
  return o;
}

// Warp `warp` of n: the run's stored elements (of the output or of a part) that
// are NaN though their row's weights are not become what the non-finite elements
// that the row sees sum to, if there are any.
template <typename T, int D, int RG>
__device__ __noinline__ void restore(const Params& p, const Bars* bs, int warp, int n) {
  const int lane = threadIdx.x & 31;
  Walk<RG> walk(p, bs->r0, bs->req0, bs->base0, bs->u0, bs->u1);
  Seg s;
  while (walk.next(p, s)) {
    float* part = p.part + ((int64_t)blockIdx.x * 2 + (s.first ? 0 : 1)) * part_floats<D>(RG);
    for (int row = warp; row < s.rows; row += n) {
      const int rq = s.row0 + row, node = rq / p.G, hq = s.hk * p.G + rq - node * p.G;
      const int t = walk.q.cu0 + node;
      const float l = s.whole ? p.lse[(int64_t)t * p.H + hq] : part[RG * D + 2 * row + 1];
      if (l != l) continue;
      const int64_t at = (int64_t)t * p.out_st + hq * p.out_sh;
      float* f = !s.whole ? part + row * D : p.out_f32 ? reinterpret_cast<float*>(p.out) + at : nullptr;
      T* h = reinterpret_cast<T*>(p.out) + at;
#pragma unroll 1
      for (int c = lane; c < D; c += 32) {
        const float x = f ? f[c] : Elem<T>::to_f32(h[c]);
        uint32_t lost = __ballot_sync(0xffffffffu, x != x);
        while (lost) {
          const int k = __ffs(lost) - 1;
          lost &= lost - 1;
          const float y = seen_sum<T>(p, walk.r, t, walk.q.ctx, s.t0 * kBN,
                                      min(walk.q.end, s.t1 * kBN), s.hk, c - lane + k);
          if (lane != k || isfinite(y)) continue;
          if (f) f[c] = y;
          else h[c] = Elem<T>::from_f32(y);
        }
      }
    }
  }
}

// ======================================================================
// tree_kernel: groups of more than 64 rows.  One CTA an SM, 640 threads.
//   warp 0      TMA producer: K and V tiles of 128 positions, each made of
//               boxes of p.box rows (a power of two up to 128 that divides
//               the page), through two rings; the lanes issue a
//               tile's boxes side by side.  Boxes behind the last position
//               or without a page start outside the tensor: zeros.
//   warps 1, 3  lane 0 issues the MMAs of stream 0 / 1; warp 1 owns TMEM.
//   warp 2      cleans V.
//   warps 4-11  softmax stream 0, warps 12-19 stream 1: thread = row and half
//               of each tile's positions.  16 warps, since the chain of a tile
//               (QK, exponentials, PV) is longer than its parts: with 8 warps
//               of whole rows it took 7400 clocks for 256 rows.
// Each stream has its own scores S_X (128 TMEM columns, overwritten in place
// by the weights P_X) and output O_X: S_X = Q K^T, O_X += P_X V, both M128.
// One thread issues a stream's MMAs, which execute in that order: the QK that
// overwrites P_X follows the PV that reads it without waiting for its end.
// P is split into a 16-bit value and a 16-bit remainder (two MMAs), ~16
// significant bits (fp16: down to 2^-32 of a row's largest, see kLift): one
// 16-bit P would cost up to 2^-9 |v|, as much as the output's own rounding.
// Sums, maxima and O are fp32.
//
// Row groups of more than 128 rows (QT = 2): stream X takes query tile X and
// both take every K/V tile.  Smaller ones: both streams share the query tile
// and take every second K/V tile; the two are joined at the end of a segment.
//
// What bounds it: the chain of a tile (scores 0.6k clocks, weights 2.2k, PV and
// the next QK 1.8k of queueing behind the other stream's, waits 0.8k) repeats
// every 5.4k clocks a stream, the tensor pipe is busy 47 % of the time (its 48
// MMAs take 3.1k) and the exponentials without the chain would fit into 2.0k.
// 4 requests of 64 nodes on 65535 positions, 32 / 8 heads of 128, bf16: 428 to
// 450 us, 611 to 642 TFLOP/s of the two products (half more with the
// remainders').  Steps, in us there: 8 softmax warps polling issuer 583; 16
// warps 552; turns 479; PV from half of P 468; turn passed on halfway 453; waits
// without a suspend hint 438 (442 with).  Tried: dropping the remainders 380,
// but one bf16 P is 2^-9 off; exponentials taken out altogether 468 (469 then):
// they are not the limit; polling instead of suspended waits 474 (469).
template <typename T, int D, int QT, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) tree_kernel(const __grid_constant__ Params p) {
  using Gm = Geom<D, QT, PAIR>;
  constexpr int RG = 128 * QT;             // rows of a group
  constexpr bool kBf16 = Elem<T>::kDtype == HALO_DTYPE_BF16;
  extern __shared__ __align__(1024) unsigned char smem[];
  Bars* bs = reinterpret_cast<Bars*>(smem + Gm::kOffBar);
  float* sm_mx = reinterpret_cast<float*>(smem + Gm::kOffMl);   // [stream][half][128]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&bs->q_full[0], 16);
    for (int i = 0; i < 6; ++i) {
      mbar_init(&bs->k_full[i], 1);
      mbar_init(&bs->k_empty[i], 2);
      mbar_init(&bs->v_full[i], 1);
      mbar_init(&bs->v_ready[i], 1);
      mbar_init(&bs->v_empty[i], 2);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bs->s_full[x], 1);
      mbar_init(&bs->p_full[2 * x], 8);
      mbar_init(&bs->p_full[2 * x + 1], 8);
      mbar_init(&bs->turn[x], 8);
      mbar_init(&bs->pv_done[x], 1);
      mbar_init(&bs->mma_done[x], 1);
    }
    bs->abort_flag = bs->odd = 0;
    fence_mbar_init();
    prefetch_map(&p.kmap);
    prefetch_map(&p.vmap);
  }
  if (warp == 1) {
    umma::tmem_alloc(&bs->tmem_base, kTmemCols);
    umma::tmem_relinquish();
  }
  grid_dep_wait();                         // the caller's writes are visible

  int64_t u0, u1, U;
  find_run<RG, kThreads>(p, bs, u0, u1, U);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = bs->tmem_base;
  if (threadIdx.x == 0) write_desc<RG>(p, bs, u0, U);
  grid_dep_trigger();

  const uint32_t sQ = smem_addr(smem + Gm::kOffQ);
  const uint32_t sK = smem_addr(smem + Gm::kOffK);
  const uint32_t sV = smem_addr(smem + Gm::kOffV);
  constexpr int SK = Gm::kStK, SV = Gm::kStV;

  // the swizzled tiles need 1024-byte alignment, which dynamic shared memory
  // without static shared memory before it has
  const bool aligned = (sQ & 1023) == 0;
  if (!aligned && threadIdx.x == 0)
    set_device_error(p.err, static_cast<unsigned int>(-HALO_ERR_MISALIGNED));

  // Register split: 128 x 56 + 512 x 104 <= 640 x 96, the launch budget.
  if (u0 < u1 && aligned) {
  if (warp < 4) {
    umma::regs_dec<56>();
    Walk<RG> walk(p, bs->r0, bs->req0, bs->base0, u0, u1);
    Seg s;
    if (warp == 0) {
      produce<RG, Gm, true, 3>(p, bs, smem, walk);
    } else if (warp & 1) {
      // -------------------------------------------------------- MMA issuer X
      if (lane == 0) {
        const int x = warp >> 1;
        constexpr uint32_t kIdQK = umma::instr_desc_f16(128, kBN, kBf16, false, false);
        constexpr uint32_t kIdPV = umma::instr_desc_f16(128, D, kBf16, false, true);
        const uint64_t qdesc0 = umma::smem_desc_sw128(sQ, 16, 1024);
        const uint64_t kdesc0 = umma::smem_desc_sw128(sK, 16, Gm::kGroup);
        const uint64_t vdesc0 = umma::smem_desc_sw128(sV, Gm::kNextBlock, Gm::kGroup);
        const uint32_t pc = tmem + x * 128, oc = tmem + Gm::kColO + x * D;
        int g0 = 0, si = 0, j = 0;            // tiles before the segment; segments; P waits
        bool ok = true;
        while (ok && walk.next(p, s)) {
          const bool two = s.rows > 128;
          const int n = s.t1 - s.t0, step = two ? 1 : 2;
          const int nx = two ? n : (x ? n / 2 : (n + 1) / 2);
          const uint64_t qd0 = qdesc0 + (uint64_t)(((two ? x : 0) * Gm::kTileBytes) >> 4);
          int g = g0 + (two ? 0 : x);
          auto k_landed = [&](int t) {
            return wait_bar(&bs->k_full[t % SK], (t / SK) & 1, bs, p.err);
          };
          auto qk = [&](int t) {              // S_X = Q K(t)^T, K(t) has landed
            const int ik = t % SK;
            const uint64_t qd = opaque(qd0);
            const uint64_t kd = opaque(kdesc0 + (uint64_t)((ik * Gm::kTileBytes) >> 4));
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              umma::mma_ss(pc, qd + (((kk >> 2) * Gm::kBlockBytes + (kk & 3) * 32) >> 4),
                           kd + (((kk >> 2) * Gm::kNextBlock + (kk & 3) * 32) >> 4), kIdQK, kk > 0);
            }
            umma::commit(&bs->s_full[x]);
            umma::commit(&bs->k_empty[ik]);
          };
          // every segment is seen by both issuers, and its end waits for both:
          // q_full cannot come round while one of them has yet to look
          ok = wait_bar(&bs->q_full[0], si & 1, bs, p.err);
          if (nx == 0) umma::commit(&bs->pv_done[x]);
          if (ok && nx > 0) ok = k_landed(g);
          if (ok && nx > 0) {
            umma::fence_after_sync();
            qk(g);
          }
          for (int it = 0; ok && it < nx; ++it, ++j) {
            const int iv = g % SV;
            // everything but P is waited for ahead of it: the next QK follows
            // this PV at once
            ok = wait_bar(&bs->v_ready[iv], (g / SV) & 1, bs, p.err) &&
                 (it + 1 == nx || k_landed(g + step));
            const uint64_t vd = opaque(vdesc0 + (uint64_t)((iv * Gm::kTileBytes) >> 4));
#pragma unroll
            for (int c = 1; c >= 0; --c) {          // O_X += P_X V(g), as the halves of P come
              ok = ok && wait_bar(&bs->p_full[2 * x + c], j & 1, bs, p.err);
              if (!ok) break;
              umma::fence_after_sync();
#pragma unroll
              for (int kk = 0; kk < 8; ++kk) {      // 16 positions: values, remainders
                const int h = kk >> 2, b = (kk >> 1) & 1;
                umma::mma_ts(oc, pc + h * 64 + c * 32 + (kk & 1) * 16 + b * 8,
                             vd + (uint64_t)(((h * 4 + c * 2 + b) * 2 * Gm::kGroup) >> 4), kIdPV,
                             it > 0 || c == 0 || kk > 0);
              }
            }
            if (!ok) break;
            g += step;
            if (it + 1 < nx) qk(g);
            else umma::commit(&bs->pv_done[x]);
            umma::commit(&bs->v_empty[iv]);
          }
          g0 += n;
          ++si;
        }
        // this thread's MMAs complete before the CTA can free TMEM
        umma::commit(&bs->mma_done[x]);
        mbar_wait(&bs->mma_done[x], 0, p.err);
      }
    } else {
      clean<T, D, RG, Gm>(p, bs, smem, walk, [] { return true; });
    }
  } else {
    umma::regs_inc<104>();
    // ------------------------------------------------------------ softmax
    // Thread: row r of stream x's scores, positions [64 h, 64 h + 64) of each
    // tile.  Both halves of a row keep one maximum.
    const int x = (warp - 4) >> 3, h = ((warp - 4) >> 2) & 1;
    const int sub = warp & 3, r = sub * 32 + lane;       // TMEM lane
    const int tid = threadIdx.x - 128;                   // 0..511
    const uint32_t trow = tmem + ((uint32_t)(sub * 32) << 16);
    const uint32_t scol = trow + x * 128 + h * 64;
    Walk<RG> walk(p, bs->r0, bs->req0, bs->base0, u0, u1);
    Seg s;
    int j = 0, si = 0;                     // this stream's tiles; segments
    int turns = 0;                         // waited for
    bool ok = true;
    while (walk.next(p, s)) {
      const bool two = QT == 2 && s.rows > 128;
      const int nodes = walk.q.nodes, ctx = walk.q.ctx, end = walk.q.end, cu0 = walk.q.cu0;
      // ---- Q: the previous segment's MMAs and scratch are done with
      named_bar_sync(1, 512);
      {
        constexpr int VPR = D / 8;
        const T* qb = reinterpret_cast<const T*>(p.q) + (int64_t)cu0 * p.q_st +
                      (int64_t)s.hk * p.G * p.q_sh;
        for (int i = tid; i < (two ? 256 : 128) * VPR; i += 512) {
          const int row = i / VPR, c = i % VPR, q = row & 127;
          const int rq = s.row0 + row, node = rq / p.G;
          const bool in = row < s.rows;
          copy16(sQ + (row >> 7) * Gm::kTileBytes + (c >> 3) * Gm::kBlockBytes + q * 128 +
                     (((c & 7) ^ (q & 7)) << 4),
                 in ? qb + node * p.q_st + (rq - node * p.G) * p.q_sh + c * 8 : qb, in);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bs->q_full[0]);
      }
      const int n = s.t1 - s.t0, step = two ? 1 : 2;
      const int n1 = two ? n : n / 2;                    // tiles of stream 1
      const int nx = x ? n1 : (two ? n : (n + 1) / 2);
      const int ny = x ? (two ? n : (n + 1) / 2) : n1;   // of the other stream
      const int rowx = s.row0 + (two ? x * 128 : 0);     // request row of lane 0
      const int rows = min(s.row0 + s.rows - rowx, 128);
      const int node = (rowx + r) / p.G;                 // of this thread's row
      float m = kNoMax, l = 0.f;
      for (int it = 0; it < nx; ++it, ++j) {
        const int p0 = (s.t0 + (two ? 0 : x) + it * step) * kBN + h * 64;
        // which of the thread's positions its row sees
        const bool full = p0 + 64 <= ctx;
        uint32_t vis[2];
        if (!full) {
          // a lane a position: positions of the context, and of the nodes
          bool context[2], drafted[2];
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int pos = p0 + 32 * w + lane;
            context[w] = pos < ctx;
            drafted[w] = pos >= ctx && pos < end;
            vis[w] = __ballot_sync(0xffffffffu, context[w]);
          }
          if (__any_sync(0xffffffffu, drafted[0] || drafted[1])) {
            // the warp's rows are those of a few consecutive nodes: one mask
            // row at a time, eight in flight
            const int n0 = __shfl_sync(0xffffffffu, node, 0);
            const int n1 = min(__shfl_sync(0xffffffffu, node, 31) + 1, nodes);
            const uint8_t* mp = p.mask + (int64_t)(cu0 + n0) * p.mask_stride + (p0 + lane - ctx);
#pragma unroll 1
            for (int k = n0; k < n1; k += 8) {
              uint8_t b[8][2];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
#pragma unroll
                for (int w = 0; w < 2; ++w)
                  b[e][w] = drafted[w] && k + e < n1 ? mp[e * p.mask_stride + 32 * w] : 0;
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) {
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                  const uint32_t bits = __ballot_sync(0xffffffffu, b[e][w] != 0);
                  if (node == k + e) vis[w] |= bits;
                }
              }
              mp += 8 * p.mask_stride;
            }
          }
        }
        ok = ok && __all_sync(0xffffffffu, wait_bar(&bs->s_full[x], j & 1, bs, p.err));
        // The streams take turns, 0 first, so that one's softmax runs beside
        // the other's MMAs: left alone they fall into step, both softmaxes and
        // then both streams' MMAs (7000 clocks for 256 rows).
        if (x == 1 || (it > 0 && it <= ny)) {
          ok = ok && __all_sync(0xffffffffu, wait_bar(&bs->turn[x], turns & 1, bs, p.err));
          ++turns;
        }
        umma::fence_after_sync();
        // 32 positions at a time, read once for the maximum and again for the
        // weights: 64 of them held would spill.  The second 32 are weighed
        // first, from the registers that their maximum left.
        float sv[32];
        auto scores = [&](int c) {
          umma::tmem_ld32(scol + c * 32, sv);
          umma::tmem_wait_ld();
          if (!full) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((vis[c] >> e) & 1u)) sv[e] = -INFINITY;
          }
        };
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          scores(c);
          float mx4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) mx4[e] = fmaxf(sv[e], sv[4 + e]);
#pragma unroll
          for (int e = 8; e < 32; ++e) {
            if ((e & 4) == 0) mx4[e & 3] = fmax3(mx4[e & 3], sv[e], sv[e + 4]);
          }
          mx = fmaxf(mx, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])));
        }
        // the maximum moves only past its headroom (weights are at most 2^8,
        // lifted 2^15), for both halves of a row at once
        bool rise = it == 0;
        if (it > 0) rise = vote_bar<256>(2 + x, rises(mx, m, p.headroom));
        if (rise) {
          sm_mx[(x * 2 + h) * 128 + r] = mx;
          named_bar_sync(2 + x, 256);
          mx = fmaxf(mx, sm_mx[(x * 2 + 1 - h) * 128 + r]);
          const bool grow = rises(mx, m, p.headroom);
          const float fac = grow ? ex2(excess(m, mx) * p.scale_log2) : 1.f;
          m = grow ? mx : m;
          l *= fac;
          if (it > 0) {
            // this half's columns of O_X, which is quiescent: the last PV was
            // issued before this QK, so it has completed, and the next PV
            // waits for this P
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
              float ov[16];
              const uint32_t oc = trow + Gm::kColO + x * D + h * (D / 2) + c;
              tmem_ld(oc, ov);
              umma::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) ov[e] *= fac;
              tmem_st(oc, ov);
            }
          }
        }
        const uint64_t sc2 = f2pack(p.scale_log2, p.scale_log2), nm2 = f2pack(-m, -m);
        uint64_t rs2 = 0;
#pragma unroll
        for (int c = 1; c >= 0; --c) {     // 16 columns of values, 16 of remainders
          if (c == 0) scores(0);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              rs2 = fadd2(rs2, weigh<T>(sv[b * 16 + 2 * e], sv[b * 16 + 2 * e + 1], sc2, nm2, hi[e],
                                        lo[e]));
            tmem_st8u(scol + c * 32 + b * 8, hi);
            tmem_st8u(scol + c * 32 + 16 + b * 8, lo);
          }
          umma::tmem_wait_st();
          umma::fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bs->p_full[2 * x + c]);
            // passed on halfway: the other stream's scores are read meanwhile
            if (c == 1 && (x == 0 ? it < ny : it + 1 < ny)) mbar_arrive(&bs->turn[1 - x]);
          }
        }
        float rs0, rs1;
        f2unpack(rs2, rs0, rs1);
        l += rs0 + rs1;
      }

      // ---- epilogue.  Named barriers are passed whether or not a wait
      // failed, so that no thread is left behind at one.  Both streams'
      // products are done before the query tile's space is scratch.
      ok = ok && __all_sync(0xffffffffu, wait_bar(&bs->pv_done[0], si & 1, bs, p.err));
      ok = ok && __all_sync(0xffffffffu, wait_bar(&bs->pv_done[1], si & 1, bs, p.err));
      umma::fence_after_sync();
      float* sm_l = reinterpret_cast<float*>(smem + Gm::kOffQ);   // [stream][half][128]
      float* sm_m = sm_l + 512;                                   // [stream][128]
      sm_l[(x * 2 + h) * 128 + r] = l;
      if (h == 0) sm_m[x * 128 + r] = m;
      named_bar_sync(1, 512);
      const bool fix = *reinterpret_cast<volatile int*>(&bs->bad[si % kBadSlots]) != 0;
      float* part = p.part + ((int64_t)blockIdx.x * 2 + (s.first ? 0 : 1)) * part_floats<D>(RG);
      auto bad = [&](int row, int col) {
        return bad_sum<T>(p, walk.r, cu0 + (s.row0 + row) / p.G, ctx, max(ctx, s.t0 * kBN),
                          min(end, s.t1 * kBN), s.hk, col);
      };
      float odd = 0.f;                     // NaN if any element is not finite
      // N columns from col of a row of the group: o scaled by 1 / L, or as it
      // is to the workspace
      auto store = [&](int row, int col, float M, float L, auto& o) {
        constexpr int N = sizeof(o) / sizeof(float);
        if (fix)
          for (int e = 0; e < N; ++e) o[e] += bad(row, col + e);
#pragma unroll
        for (int e = 0; e < N; ++e) odd = fmaf(o[e], 0.f, odd);
        if (!s.whole) {
          float4* d = reinterpret_cast<float4*>(part + row * D + col);
#pragma unroll
          for (int e = 0; e < N; e += 4) d[e / 4] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          if (col == 0) *reinterpret_cast<float2*>(part + RG * D + 2 * row) = make_float2(M, L);
          return;
        }
        const int rq = s.row0 + row, node = rq / p.G, hq = s.hk * p.G + rq - node * p.G;
        const int64_t t = cu0 + node;
        const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
        if (col == 0)
          p.lse[t * p.H + hq] = log_sum<T>(M, L, p.scale_log2);
        const int64_t at = t * p.out_st + hq * p.out_sh + col;
        if (p.out_f32) {
          float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at);
#pragma unroll
          for (int e = 0; e < N; e += 4)
            d[e / 4] = make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
        } else {
          uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + at);
#pragma unroll
          for (int e = 0; e < N; e += 8)
            d[e / 8] = make_uint4(Elem<T>::pack(o[e] * inv, o[e + 1] * inv),
                                  Elem<T>::pack(o[e + 2] * inv, o[e + 3] * inv),
                                  Elem<T>::pack(o[e + 4] * inv, o[e + 5] * inv),
                                  Elem<T>::pack(o[e + 6] * inv, o[e + 7] * inv));
        }
      };
      if (two) {
        // stream x's rows, half the columns a thread
        const float L = sm_l[x * 256 + r] + sm_l[x * 256 + 128 + r];
#pragma unroll 1
        for (int c = 0; c < D / 2; c += 16) {
          float ov[16];
          tmem_ld(trow + Gm::kColO + x * D + h * (D / 2) + c, ov);
          umma::tmem_wait_ld();
          if (r < rows && ok) store(r + x * 128, h * (D / 2) + c, m, L, ov);
        }
      } else {
        // the two streams' states of a row are both in its TMEM lane: every
        // thread joins a quarter of the columns.  A state that saw nothing has
        // l = 0 and o = 0 beside kNoMax, one that saw only NaN l = NaN: either
        // joins right with any weight.
        const float m0 = sm_m[r], m1 = n1 > 0 ? sm_m[128 + r] : kNoMax;
        const float l0 = sm_l[r] + sm_l[128 + r], l1 = n1 > 0 ? sm_l[256 + r] + sm_l[384 + r] : 0.f;
        const float M = fmaxf(m0, m1);
        const float w0 = join_weight(m0, M, p.scale_log2), w1 = join_weight(m1, M, p.scale_log2);
        const float L = fmaf(l1, w1, l0 * w0);
        const int col = (x * 2 + h) * (D / 4);
#pragma unroll 1
        for (int c = 0; c < D / 4; c += 16) {
          float a[16], b[16];
          tmem_ld(trow + Gm::kColO + col + c, a);
          if (n1 > 0) tmem_ld(trow + Gm::kColO + D + col + c, b);
          umma::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) a[e] = n1 > 0 ? fmaf(b[e], w1, a[e] * w0) : a[e] * w0;
          if (r < rows && ok) store(r, col + c, M, L, a);
        }
      }
      if (odd != odd) bs->odd = 1;
      umma::fence_before_sync();
      ++si;
    }
    // by these warps alone: the others gave registers away that the call may use
    named_bar_sync(1, 512);
    if (bs->odd) restore<T, D, RG>(p, bs, warp - 4, 16);
  }
  }

  // ---- teardown: every TMEM access and MMA has completed
  umma::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    umma::fence_after_sync();
    umma::tmem_dealloc(tmem, kTmemCols);
  }
}

// ======================================================================
// tree_few_kernel: groups of at most 64 rows (NR = 16, 32 or 64).  One CTA an
// SM, 416 threads (NR < 64), 384 or 640.
//   warp 0      TMA producer (as in tree_kernel); the last warp of 416 threads
//               V's
//   warps 1, 3  lane 0 issues the QK / PV MMAs (one thread for both took 1950
//               clocks a tile, most of them in commits); warp 1 owns TMEM
//   warp 2      cleans V; query rows of the next segment (two buffers; the
//               first segment's are loaded by the softmax warps)
//   from 4      softmax (thread = position of the tile) and epilogue (thread =
//               output column), four warps for each NR / kGroups rows
// Both products have the K/V tile as the 128-row operand and the query rows
// as the columns: S^T = K Q^T (M = positions, N = NR) and O^T += V^T P^T
// (M = columns of V, N = 2 NR: the weights' 16-bit values and, beside them,
// their 16-bit remainders, so V goes through the tensor pipe once).  With the
// rows on the 128-row side, as in tree_kernel, the MMAs of 8 rows would cost
// the energy of 128, and what bounds a long context is the clock that the
// power limit leaves beside the memory's own draw: one request of a million
// tokens ran at 1.33 GHz that way.  An MMA takes 60 to 70 clocks for any N up
// to 128 (its 4 KB of K or V from shared memory), 1000 a tile, well under the
// 2800 that the tile's bytes take at 1.9 GHz.
// The row maximum lies across threads here, but it moves only past its
// headroom of 2^8, so a tile costs one barrier with a vote; the reduction runs
// in a segment's first tile and in the rare tile that raises it.
//
// What it reaches: 1M positions, 64 / 8 heads of 128, 4 nodes (4.3 GB): 616 to
// 704 us by the clock that the power limit leaves, 6.1 to 7.0 TB/s (a plain copy
// 6.5); with rows on the 128-row side 899.  8 requests of 16 nodes on 32768
// positions (1.08 GB): 213 to 233 us, 4.6 to 5.1 TB/s: 192 us for the tiles of an
// SM, 4 before the first, 3 for an epilogue, 4 for a second segment, 4 for the
// merge and the launch.  One softmax group of all rows: 248; parts in rows of
// 528 bytes: 225.  At 64 columns a tile's bytes take 1.4k clocks, the chain of
// its softmax more: 8 requests on 32768 positions (82 us of bytes) take 99 us
// with 16 rows, 120 with 32, 145 to 154 with 64.  Small batches are latency: 10 us
// for one token on 1000 positions (find the run 1.1, first rows and tables 1.5,
// first tile 1.5, softmax and PV 1.9, epilogue 1.1, merge 3).

// Sum or maximum over the warp of N (8, 16 or 32) columns, one a row: lane i
// ends with row i % N in v[0].
template <int N, class Op>
__device__ __forceinline__ void warp_columns(float (&v)[N], Op op) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o >= N; o >>= 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = op(v[i], __shfl_xor_sync(0xffffffffu, v[i], o));
  }
#pragma unroll
  for (int o = N / 2; o >= 1; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = up ? v[i + o] : v[i], give = up ? v[i] : v[i + o];
      v[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, o));
    }
  }
}

template <typename T, int D, int NR, bool PAIR>
__global__ void __launch_bounds__(FewGeom<D, NR, PAIR>::kThreads, 1)
    tree_few_kernel(const __grid_constant__ Params p) {
  using Gm = FewGeom<D, NR, PAIR>;
  constexpr int RG = NR;
  constexpr bool kBf16 = Elem<T>::kDtype == HALO_DTYPE_BF16;
  constexpr int SK = Gm::kStK, SV = Gm::kStV, PB = Gm::kPBuf;
  constexpr uint32_t kCols = 4 * NR;             // TMEM: S twice, O
  extern __shared__ __align__(1024) unsigned char smem[];
  Bars* bs = reinterpret_cast<Bars*>(smem + Gm::kOffBar);
  FewShared* sh = reinterpret_cast<FewShared*>(smem + Gm::kOffRed);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bs->q_full[i], 1);
      mbar_init(&bs->q_empty[i], 1);
      mbar_init(&bs->s_full[i], 1);
      mbar_init(&bs->s_free[i], Gm::kSoft / 32);
    }
    for (int i = 0; i < 6; ++i) {
      mbar_init(&bs->k_full[i], 1);
      mbar_init(&bs->k_empty[i], 1);
      mbar_init(&bs->v_full[i], 1);
      mbar_init(&bs->v_ready[i], 1);
      mbar_init(&bs->v_empty[i], 1);
    }
    mbar_init(&bs->p_full[0], Gm::kSoft / 32);
    mbar_init(&bs->p_full[1], Gm::kSoft / 32);
    mbar_init(&bs->pv_done[0], 1);
    mbar_init(&bs->pv_done[1], 1);
    mbar_init(&bs->mma_done[0], 1);
    mbar_init(&bs->mma_done[1], 1);
    bs->abort_flag = bs->odd = 0;
    fence_mbar_init();
    prefetch_map(&p.kmap);
    prefetch_map(&p.vmap);
  }
  if (warp == 1) {
    umma::tmem_alloc(&bs->tmem_base, kCols);
    umma::tmem_relinquish();
  }
  grid_dep_wait();                         // the caller's writes are visible
  int64_t u0, u1, U;
  find_run<RG, Gm::kThreads>(p, bs, u0, u1, U);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = bs->tmem_base;
  if (threadIdx.x == 64) write_desc<RG>(p, bs, u0, U);
  grid_dep_trigger();

  const uint32_t sQ = smem_addr(smem + Gm::kOffQ);
  const uint32_t sK = smem_addr(smem + Gm::kOffK);
  const uint32_t sV = smem_addr(smem + Gm::kOffV);
  const uint32_t sP = smem_addr(smem + Gm::kOffP);
  const bool aligned = (sK & 1023) == 0;   // as in tree_kernel
  if (!aligned && threadIdx.x == 0)
    set_device_error(p.err, static_cast<unsigned int>(-HALO_ERR_MISALIGNED));

  if (u0 < u1 && aligned) {
    Walk<RG> walk(p, bs->r0, bs->req0, bs->base0, u0, u1);
    Seg s;
    // Segment si's query rows by threads 0 .. nt - 1: 16-byte copies, all in
    // flight.
    auto copy_q = [&](const Walk<RG>& w, const Seg& s, int t, int nt, int si) {
      constexpr int VPR = D / 8;
      const char* qb = p.q + 2 * (w.q.cu0 * p.q_st + (int64_t)s.hk * p.G * p.q_sh);
      const uint32_t dst = sQ + (si & 1) * Gm::kQBytes;
#pragma unroll 1
      for (int i = t; i < NR * VPR; i += nt) {
        const int row = i / VPR, c = i % VPR;
        const int rq = s.row0 + row, node = rq / p.G;
        const bool in = row < s.rows;
        const char* src = qb + 2 * (node * p.q_st + (rq - node * p.G) * p.q_sh + c * 8);
        copy16(dst + (c >> 3) * NR * 128 + row * 128 + (((c & 7) ^ (row & 7)) << 4),
               in ? src : p.q, in);
      }
    };
    if (warp == 0) {
      produce<RG, Gm, false, NR == 64 ? 3 : 1>(p, bs, smem, walk);
    } else if (NR < 64 && warp == 4 + Gm::kSoft / 32) {
      produce<RG, Gm, false, 2>(p, bs, smem, walk);
    } else if (warp == 1) {
      // -------------------------------------------------------- QK issuer
      if (lane == 0) {
        constexpr uint32_t kIdQK = umma::instr_desc_f16(kBN, NR, kBf16, false, false);
        const uint64_t kdesc0 = umma::smem_desc_sw128(sK, 16, Gm::kGroup);
        int g = 0, si = 0;                  // tiles; segments
        bool ok = true;
        while (ok && walk.next(p, s)) {
          const uint64_t qd0 = umma::smem_desc_sw128(sQ + (si & 1) * Gm::kQBytes, 16, 1024);
          ok = wait_bar(&bs->q_full[si & 1], (si >> 1) & 1, bs, p.err);
          for (int t = s.t0; ok && t < s.t1; ++t, ++g) {   // S^T = K(g) Q^T
            const int ik = g % SK;
            ok = wait_bar(&bs->k_full[ik], (g / SK) & 1, bs, p.err) &&
                 (g < 2 || wait_bar(&bs->s_free[g & 1], ((g >> 1) - 1) & 1, bs, p.err));
            if (!ok) break;
            umma::fence_after_sync();
            const uint64_t qd = opaque(qd0);
            const uint64_t kd = opaque(kdesc0 + (uint64_t)((ik * Gm::kTileBytes) >> 4));
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              umma::mma_ss(tmem + (g & 1) * NR,
                           kd + (uint64_t)(((kk >> 2) * Gm::kNextBlock + (kk & 3) * 32) >> 4),
                           qd + (uint64_t)(((kk >> 2) * NR * 128 + (kk & 3) * 32) >> 4), kIdQK,
                           kk > 0);
            umma::commit(&bs->s_full[g & 1]);
            umma::commit(&bs->k_empty[ik]);
          }
          umma::commit(&bs->q_empty[si & 1]);
          ++si;
        }
        umma::commit(&bs->mma_done[0]);
        mbar_wait(&bs->mma_done[0], 0, p.err);
      }
    } else if (warp == 3) {
      // -------------------------------------------------------- PV issuer
      if (lane == 0) {
        constexpr uint32_t kIdPV = umma::instr_desc_f16(128, 2 * NR, kBf16, true, true);
        // V^T has 128 rows; 64 columns of V fill them twice (the same block
        // again), and the second half of O^T is not read
        const uint64_t vdesc0 =
            umma::smem_desc_sw128(sV, D == 64 ? 0 : Gm::kNextBlock, Gm::kGroup);
        const uint64_t pdesc0 = umma::smem_desc_sw128(sP, Gm::kBlockBytes, 1024);
        int g = 0;
        bool ok = true;
        while (ok && walk.next(p, s)) {
          for (int t = s.t0; ok && t < s.t1; ++t, ++g) {   // O^T += V(g)^T P^T
            const int iv = g % SV;
            ok = wait_bar(&bs->v_ready[iv], (g / SV) & 1, bs, p.err) &&
                 wait_bar(&bs->p_full[g % PB], (g / PB) & 1, bs, p.err);
            if (!ok) break;
            umma::fence_after_sync();
            const uint64_t vd = opaque(vdesc0 + (uint64_t)((iv * Gm::kTileBytes) >> 4));
            const uint64_t pd = opaque(pdesc0 + (uint64_t)(((g % PB) * Gm::kPBytes) >> 4));
#pragma unroll
            for (int kk = 0; kk < kBN / 16; ++kk)
              umma::mma_ss(tmem + Gm::kColO, vd + (uint64_t)((kk * 2 * Gm::kGroup) >> 4),
                           pd + (uint64_t)((kk * 16 * 128) >> 4), kIdPV, t > s.t0 || kk > 0);
            umma::commit(&bs->pv_done[g % PB]);
            umma::commit(&bs->v_empty[iv]);
          }
        }
        umma::commit(&bs->mma_done[1]);
        mbar_wait(&bs->mma_done[1], 0, p.err);
      }
    } else if (warp == 2) {
      // cleans V, and before a segment's first tile loads the next segment's
      // query rows (the first segment's are the softmax warps'): their buffer
      // was read by products that need nothing more from this warp
      Walk<RG> ahead = walk;
      Seg sa;
      bool more = ahead.next(p, sa);
      int sq = 0;
      clean<T, D, RG, Gm>(p, bs, smem, walk, [&]() {
        more = more && ahead.next(p, sa);
        ++sq;
        if (!more) return true;
        if (sq >= 2 && !__all_sync(0xffffffffu, wait_bar(&bs->q_empty[sq & 1],
                                                         ((sq >> 1) - 1) & 1, bs, p.err)))
          return false;
        copy_q(ahead, sa, lane, 32, sq);
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bs->q_full[sq & 1]);
        return true;
      });
    } else {
      // -------------------------------------------------------- softmax
      // groups of four warps, each RT of the NR rows; thread = position
      constexpr int RT = NR / Gm::kGroups;
      const int sub = warp & 3, grp = (warp - 4) >> 2, bar = 1 + grp;
      const int tid = threadIdx.x & 127, r0 = grp * RT;
      const uint32_t trow = tmem + ((uint32_t)(sub * 32) << 16);
      int g = 0, si = 0;
      bool ok = true;
      auto pv_waited = [&](int t) {        // P V of tile t is done
        return __all_sync(0xffffffffu, wait_bar(&bs->pv_done[t % PB], (t / PB) & 1, bs, p.err));
      };
      while (walk.next(p, s)) {
        const int ctx = walk.q.ctx, end = walk.q.end;
        if (si == 0) {                     // later ones come from warp 2, ahead
          copy_q(walk, s, threadIdx.x - 128, Gm::kSoft, 0);
          asm volatile("cp.async.wait_all;" ::: "memory");
          fence_proxy_async_smem();
          named_bar_sync(1 + Gm::kGroups, Gm::kSoft);
          if (threadIdx.x == 128) mbar_arrive(&bs->q_full[0]);
        }
        float l[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) l[r] = 0.f;
        for (int t = s.t0; t < s.t1; ++t, ++g) {
          // rows that see this thread's position
          const bool full = (t + 1) * kBN <= ctx;
          uint32_t vis = 0;                // a bit a row
          if (!full) {
            const int pos = t * kBN + tid, jn = pos - ctx;
            vis = pos < ctx ? 0xffffffffu : 0u;
            if (jn >= 0 && pos < end) {
              // the nodes of this group's rows that see node jn, eight loads
              // in flight, then a bit for each of their rows
              const int first = s.row0 + r0, n0 = first / p.G;
              const int n1 = min((first + RT - 1) / p.G + 1, walk.q.nodes);
              const uint8_t* mp = p.mask + (walk.q.cu0 + n0) * p.mask_stride + jn;
              uint32_t sees = 0;
#pragma unroll 1
              for (int k = 0; k < RT && n0 + k < n1; k += 8) {
                uint8_t b[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  b[e] = n0 + k + e < n1 ? *mp : 0;
                  mp += p.mask_stride;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) sees |= (b[e] != 0 ? 1u : 0u) << (k + e);
              }
              int rem = first - n0 * p.G;
#pragma unroll
              for (int r = 0; r < RT; ++r) {
                vis |= (sees & 1u) << r;
                if (++rem == p.G) {
                  rem = 0;
                  sees >>= 1;
                }
              }
            }
          }
          ok = ok && __all_sync(0xffffffffu, wait_bar(&bs->s_full[g & 1], (g >> 1) & 1, bs, p.err));
          umma::fence_after_sync();
          // Excess of the scores over the running maxima; where a row's maximum
          // has to rise (always in the first tile) the raw scores are reduced
          // and the loop runs again, at most once a tile: it ends after three
          // passes whatever the scores are.
          float x[RT];
          bool rise = t == s.t0, risen = false;
          while (true) {
            tmem_ld(trow + (g & 1) * NR + r0, x);
            umma::tmem_wait_ld();
            if (!full) {
#pragma unroll
              for (int r = 0; r < RT; ++r)
                if (!((vis >> r) & 1u)) x[r] = -INFINITY;
            }
            if (!rise) {
              float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
              const uint64_t minus = f2pack(-1.f, -1.f);
#pragma unroll
              for (int r = 0; r < RT; r += 4) {
                // excess() of two rows at a time
                const float4 m = *reinterpret_cast<const float4*>(&sh->m[r0 + r]);
                f2unpack(ffma2(f2pack(m.x, m.y), minus, f2pack(x[r], x[r + 1])), x[r], x[r + 1]);
                f2unpack(ffma2(f2pack(m.z, m.w), minus, f2pack(x[r + 2], x[r + 3])), x[r + 2],
                         x[r + 3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], x[r + e]);
              }
              if (risen) break;
              rise = vote_bar<128>(
                  bar, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) > p.headroom);
              if (!rise) break;
              continue;
            }
            warp_columns<RT>(x, [](float a, float b) { return fmaxf(a, b); });
            if (lane < RT) sh->red[sub][r0 + lane] = x[0];
            named_bar_sync(bar, 128);
            if (tid < RT) {
              const int r = r0 + tid;
              const float mx = fmaxf(fmaxf(sh->red[0][r], sh->red[1][r]),
                                     fmaxf(sh->red[2][r], sh->red[3][r]));
              const float mo = t == s.t0 ? kNoMax : sh->m[r];
              const bool grow = rises(mx, mo, p.headroom);
              sh->fac[r] = grow ? ex2(excess(mo, mx) * p.scale_log2) : 1.f;
              sh->m[r] = grow ? mx : mo;
            }
            named_bar_sync(bar, 128);
            if (t > s.t0) {
              // O^T: every PV issued so far has to be done
              ok = ok && pv_waited(g - 1);
              umma::fence_after_sync();
              float fac[RT];
#pragma unroll
              for (int r = 0; r < RT; r += 4) {
                const float4 b = *reinterpret_cast<const float4*>(&sh->fac[r0 + r]);
                fac[r] = b.x, fac[r + 1] = b.y, fac[r + 2] = b.z, fac[r + 3] = b.w;
              }
#pragma unroll
              for (int r = 0; r < RT; ++r) l[r] *= fac[r];
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float ov[RT];
                const uint32_t oc = trow + Gm::kColO + c * NR + r0;
                tmem_ld(oc, ov);
                umma::tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < RT; ++e) ov[e] *= fac[e];
                tmem_st(oc, ov);
              }
              umma::tmem_wait_st();
            }
            rise = false;
            risen = true;
          }
          // the scores are in registers: S's buffer is free
          umma::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bs->s_free[g & 1]);
          uint32_t hi[RT / 2], lo[RT / 2];
#pragma unroll
          for (int r = 0; r < RT; r += 2) {
            float a, b;
            f2unpack(ffma2(f2pack(x[r], x[r + 1]), f2pack(p.scale_log2, p.scale_log2),
                           f2pack(kLift<T>, kLift<T>)), a, b);
            a = ex2(a);
            b = ex2(b);
            l[r] += a;
            l[r + 1] += b;
            float ah, bh;
            if constexpr (kBf16) {         // truncated: one byte permute a pair
              hi[r / 2] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
              ah = __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
              bh = __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
            } else {
              hi[r / 2] = Elem<T>::pack(a, b);
              Elem<T>::unpack(hi[r / 2], ah, bh);
            }
            lo[r / 2] = Elem<T>::pack(a - ah, b - bh);
          }
          // P's buffer is free once the PV that read it is done
          if (g >= PB) ok = ok && pv_waited(g - PB);
          // row `position` of P^T: NR values, NR remainders
          unsigned char* pr = smem + Gm::kOffP + (g % PB) * Gm::kPBytes + tid * 128;
          const int sw = tid & 7, c0 = grp * (RT / 8);
#pragma unroll
          for (int c = 0; c < RT / 8; ++c) {
            *reinterpret_cast<uint4*>(pr + (((c0 + c) ^ sw) << 4)) =
                make_uint4(hi[4 * c], hi[4 * c + 1], hi[4 * c + 2], hi[4 * c + 3]);
            unsigned char* q = NR == 64 ? pr + Gm::kBlockBytes + (((c0 + c) ^ sw) << 4)
                                        : pr + (((NR / 8 + c0 + c) ^ sw) << 4);
            *reinterpret_cast<uint4*>(q) =
                make_uint4(lo[4 * c], lo[4 * c + 1], lo[4 * c + 2], lo[4 * c + 3]);
          }
          fence_proxy_async_smem();
          umma::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bs->p_full[g % PB]);
        }

        // ---- epilogue; barriers are passed whether or not a wait failed
        ok = ok && pv_waited(g - 1);
        umma::fence_after_sync();
        warp_columns<RT>(l, [](float a, float b) { return a + b; });
        if (lane < RT) sh->red[sub][r0 + lane] = l[0];
        named_bar_sync(bar, 128);
        // where each row goes and what it is scaled by: the output, or as it
        // is to the workspace
        float* part = p.part + ((int64_t)blockIdx.x * 2 + (s.first ? 0 : 1)) * part_floats<D>(RG);
        if (tid < RT && r0 + tid < s.rows) {
          const int r = r0 + tid;
          const float L = (sh->red[0][r] + sh->red[1][r]) + (sh->red[2][r] + sh->red[3][r]);
          const float M = sh->m[r];
          if (!s.whole) {
            *reinterpret_cast<float2*>(part + RG * D + 2 * r) = make_float2(M, L);
            sh->fac[r] = 1.f;
            sh->off[r] = r * D;
          } else {
            const int rq = s.row0 + r, node = rq / p.G, hq = s.hk * p.G + rq - node * p.G;
            const int64_t row = walk.q.cu0 + node;
            p.lse[row * p.H + hq] = log_sum<T>(M, L, p.scale_log2);
            sh->fac[r] = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
            sh->off[r] = row * p.out_st + hq * p.out_sh;
          }
        }
        named_bar_sync(bar, 128);
        const bool fix = *reinterpret_cast<volatile int*>(&bs->bad[si % kBadSlots]) != 0;
        float* of = !s.whole ? part : p.out_f32 ? reinterpret_cast<float*>(p.out) : nullptr;
        float odd = 0.f;                   // NaN if any element is not finite
#pragma unroll 1
        for (int c = r0; c < min(r0 + RT, s.rows); c += 8) {
          float a[8], b[8];
          tmem_ld(trow + Gm::kColO + c, a);
          tmem_ld(trow + Gm::kColO + NR + c, b);
          float fac[8];
          int64_t off[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            fac[e] = sh->fac[c + e];
            off[e] = sh->off[c + e] + tid;
          }
          umma::tmem_wait_ld();
          if (tid >= D || !ok) continue;
#pragma unroll
          for (int e = 0; e < 8; ++e) a[e] += b[e];
          if (fix) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c + e < s.rows)
                a[e] += bad_sum<T>(p, walk.r, walk.q.cu0 + (s.row0 + c + e) / p.G, ctx,
                                   max(ctx, s.t0 * kBN), min(end, s.t1 * kBN), s.hk, tid);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) odd = fmaf(a[e], 0.f, odd);
          if (of) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c + e < s.rows) of[off[e]] = a[e] * fac[e];
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c + e < s.rows)
                reinterpret_cast<T*>(p.out)[off[e]] = Elem<T>::from_f32(a[e] * fac[e]);
          }
        }
        if (odd != odd) bs->odd = 1;
        umma::fence_before_sync();
        ++si;
      }
      named_bar_sync(1 + Gm::kGroups, Gm::kSoft);
      if (bs->odd) restore<T, D, NR>(p, bs, warp - 4, Gm::kSoft / 32);
    }
  }

  // ---- teardown: every TMEM access and MMA has completed
  umma::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    umma::fence_after_sync();
    umma::tmem_dealloc(tmem, kCols);
  }
}

// ======================================================================
// tree_merge_kernel: joins the parts of segments that were cut.  Block
// (c - 1, y) looks at the cut between CTAs c - 1 and c; the first cut inside
// a segment owns it, and its blocks share the rows, a warp a row.
// Latency-bound (about 3 us behind the attention kernel): the lanes find the
// CTAs that hold a part side by side; dividing for every cut took 8 us.
constexpr int kMergeWarps = 8;
constexpr int kMergeRowBlocks = 16;      // 8: 1 to 9 % slower with many rows, 32: empty blocks

template <typename T, int D>
__global__ void __launch_bounds__(kMergeWarps * 32) tree_merge_kernel(
    const __grid_constant__ Params p, int n_cta, int RG) {
  constexpr int C = D / 32;
  grid_dep_wait();
  grid_dep_trigger();                      // the next kernel may begin its set-up
  const int c = (int)blockIdx.x + 1;
  const Desc d = p.desc[c];
  const int lane = threadIdx.x & 31;
  int row = (int)blockIdx.y * kMergeWarps + (threadIdx.x >> 5);
  if (row >= d.rows) return;
  // the cut before CTA i, in tiles of this segment (a cut in its set-up units
  // or before it: 0); i U / n = i (U / n) + i (U mod n) / n
  auto cut = [&](int i) {
    const int64_t t = i * d.quot + (uint32_t)(i * d.rem) / (uint32_t)n_cta - d.start;
    return (int)min(max(t, (int64_t)0), (int64_t)d.nt);
  };
  const int own = cut(c);
  if (own <= 0 || own >= d.nt || cut(c - 1) > 0) return;
  const int64_t before = (c - 1) * d.quot + (uint32_t)((c - 1) * d.rem) / (uint32_t)n_cta;
  for (; row < d.rows; row += (int)gridDim.y * kMergeWarps) {
    float M = -INFINITY, L = 0.f, acc[C];
#pragma unroll
    for (int e = 0; e < C; ++e) acc[e] = 0.f;
    for (int i0 = c - 1; i0 < n_cta && cut(i0) < d.nt; i0 += 32) {
      const int a = cut(i0 + lane), b = cut(i0 + lane + 1);
      uint32_t has = __ballot_sync(0xffffffffu, i0 + lane < n_cta && a < b);
      while (has) {
        constexpr int B = 4;
        float2 ml[B];
        float o[B][C];
#pragma unroll
        for (int u = 0; u < B; ++u) {
          ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
          for (int e = 0; e < C; ++e) o[u][e] = 0.f;
          if (has) {
            const int i = i0 + __ffs(has) - 1;
            has &= has - 1;
            // CTA c - 1 may have begun before the segment's set-up units: then
            // this is its second part
            const int sl = i == c - 1 && before < d.start - (RG <= 64 ? kSetup<64> : kSetup<128>) ? 1 : 0;
            const float* s = p.part + ((int64_t)i * 2 + sl) * part_floats<D>(RG);
            ml[u] = *reinterpret_cast<const float2*>(s + RG * D + 2 * row);
            s += row * D;
            if constexpr (C == 4) {
              const float4 y = *reinterpret_cast<const float4*>(s + lane * 4);
              o[u][0] = y.x;
              o[u][1] = y.y;
              o[u][2] = y.z;
              o[u][3] = y.w;
            } else {
              const float2 y = *reinterpret_cast<const float2*>(s + lane * 2);
              o[u][0] = y.x;
              o[u][1] = y.y;
            }
          }
        }
        float Mn = M;
#pragma unroll
        for (int u = 0; u < B; ++u) Mn = fmaxf(Mn, ml[u].x);
        // a part that saw nothing or only NaN joins right with any weight (l and
        // o are 0, or l is NaN), and Mn is at least kNoMax
        const float a0 = join_weight(M, Mn, p.scale_log2);
        L *= a0;
#pragma unroll
        for (int e = 0; e < C; ++e) acc[e] *= a0;
#pragma unroll
        for (int u = 0; u < B; ++u) {
          const float w = join_weight(ml[u].x, Mn, p.scale_log2);
          L = fmaf(ml[u].y, w, L);
#pragma unroll
          for (int e = 0; e < C; ++e) acc[e] = fmaf(o[u][e], w, acc[e]);
        }
        M = Mn;
      }
    }
    const int rq = d.row0 + row, node = rq / p.G, hq = d.hk * p.G + rq - node * p.G;
    const int64_t t = d.cu0 + node;
    const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
    if (lane == 0) p.lse[t * p.H + hq] = log_sum<T>(M, L, p.scale_log2);
    const int64_t at = t * p.out_st + hq * p.out_sh + lane * C;
    if (p.out_f32) {
      float* o = reinterpret_cast<float*>(p.out) + at;
#pragma unroll
      for (int e = 0; e < C; ++e) o[e] = acc[e] * inv;
    } else {
      uint32_t* o = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + at);
#pragma unroll
      for (int e = 0; e < C; e += 2) o[e / 2] = Elem<T>::pack(acc[e] * inv, acc[e + 1] * inv);
    }
  }
}

}  // namespace tree

// ================================================================ host side
namespace tree {

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                             const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeFn encode_fn() {
  static EncodeFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(ptr);
  });
  return fn;
}

// The tensor map of a pool's K or V: {D, page, H_kv, n_pages} with boxes of 64
// columns x `box` rows or, for boxes of both column blocks, {64, page, 2,
// H_kv, n_pages} (a swizzled box is at most 128 bytes wide); 128-byte swizzle,
// zeros outside.
static int encode_pool(const halo_page_pool_t* pool, const void* ptr, int64_t stride_p,
                       int64_t stride_h, int64_t stride_t, int box, bool pair, CUtensorMap* out) {
  EncodeFn fn = encode_fn();
  if (!fn) return fail(HALO_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  // the stride of a dimension of one is never used, but has to be legal
  const cuuint64_t st = stride_t * 2;
  const cuuint64_t sh = pool->H_kv > 1 ? stride_h * 2 : st;
  const cuuint64_t sp = pool->n_pages > 1 ? stride_p * 2 : st;
  const cuuint64_t page = pool->page_size, H_kv = pool->H_kv, n_pages = pool->n_pages;
  const cuuint32_t rows = box;
  const cuuint64_t dims4[4] = {(cuuint64_t)pool->D, page, H_kv, n_pages}, str4[3] = {st, sh, sp};
  const cuuint64_t dims5[5] = {64, page, 2, H_kv, n_pages}, str5[4] = {st, 128, sh, sp};
  const cuuint32_t box4[4] = {64, rows, 1, 1}, box5[5] = {64, rows, 2, 1, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r =
      fn(out, pool->dtype == HALO_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                             : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
         pair ? 5 : 4, const_cast<void*>(ptr), pair ? dims5 : dims4, pair ? str5 : str4,
         pair ? box5 : box4, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(HALO_ERR_INVALID_ARG,
                "page pool tensor map encode failed (%d): %d pages, page %d, strides %lld %lld "
                "%lld bytes", (int)r, pool->n_pages, pool->page_size, (long long)sp, (long long)sh,
                (long long)st);
  return HALO_OK;
}

static bool rows16(const void* p, int64_t a, int64_t b, int64_t c, int elt) {
  return ((reinterpret_cast<uintptr_t>(p) | (uint64_t)(a * elt) | (uint64_t)(b * elt) |
           (uint64_t)(c * elt)) & 15) == 0;
}

// Whether two of the rows of D elements at t * st + h * sh (t < T, h < H) share
// an element: two heads dh apart and two tokens dt apart whose distances differ
// by less than D.  dt next to dh * sh / st is the nearest.
static bool rows_overlap(int64_t T, int64_t st, int64_t H, int64_t sh, int64_t D) {
  if ((T > 1 && st < D) || (H > 1 && sh < D)) return true;
  if (T <= 1 || H <= 1) return false;
  if (st / H >= sh || sh / T >= st) return false;         // one inside the other, as in a tensor
  for (int64_t dh = 1; dh < H; ++dh) {
    const int64_t dt = dh * sh / st, over = dh * sh - dt * st;   // 0 <= over < st
    if (dt >= T) return false;
    if (over < D || (dt + 1 < T && st - over < D)) return true;
  }
  return false;
}

static int check(const halo_page_pool_t* pool, const halo_tree_problem_t* pb) {
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
  if (pb->H > 65535) return fail(HALO_ERR_UNSUPPORTED, "%d heads", pb->H);
  if ((int64_t)pb->max_blocks * pool->page_size + 2048 > INT_MAX)
    return fail(HALO_ERR_UNSUPPORTED, "block tables of %d pages of %d are too long", pb->max_blocks,
                pool->page_size);
  if (!(pb->scale > 0.f) || !std::isfinite(pb->scale))
    return fail(HALO_ERR_UNSUPPORTED, "tree attention needs a positive finite scale");
  return HALO_OK;
}

// Rows of a group, from the most rows a request can have on one K/V head:
// the smallest of 16, 32, 64, 128 and 256 that holds them (256 at most).
static int group_rows(const halo_page_pool_t* pool, const halo_tree_problem_t* pb) {
  const int64_t rows = (int64_t)pb->max_nodes * (pb->H / pool->H_kv);
  return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
}

static int64_t desc_bytes(int n_cta) { return ((int64_t)n_cta * sizeof(Desc) + 255) & ~int64_t(255); }

static int64_t part_bytes(const halo_page_pool_t* pool, const halo_tree_problem_t* pb, int n_cta) {
  return (int64_t)n_cta * 2 * group_rows(pool, pb) * (pool->D + 2) * sizeof(float);
}

static int64_t ws_bytes(const halo_page_pool_t* pool, const halo_tree_problem_t* pb) {
  const int n = device_sms();
  return desc_bytes(n) + part_bytes(pool, pb, n) +
         (pb->lse ? 0 : (int64_t)pb->T * pb->H * sizeof(float));
}

template <typename T, int D, int RG, bool PAIR>
static int launch(const Params& p, int n_cta, cudaStream_t st) {
  void (*kernel)(const Params);
  int smem, threads;
  if constexpr (RG <= 64) {
    kernel = tree_few_kernel<T, D, RG, PAIR>;
    smem = FewGeom<D, RG, PAIR>::kSmemBytes;
    threads = FewGeom<D, RG, PAIR>::kThreads;
  } else {
    kernel = tree_kernel<T, D, RG / 128, PAIR>;
    smem = Geom<D, RG / 128, PAIR>::kSmemBytes;
    threads = kThreads;
  }
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63], [&] {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (e != cudaSuccess) return cuda_fail(e, "tree kernel shared-memory attribute");
  e = launch_dependent(kernel, dim3((unsigned)n_cta), dim3((unsigned)threads), (size_t)smem, st, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "tree kernel launch");
  count_launches();
  if (n_cta > 1) {
    e = launch_dependent(tree_merge_kernel<T, D>,
                         dim3((unsigned)n_cta - 1, std::min(RG / kMergeWarps, kMergeRowBlocks)),
                         dim3(kMergeWarps * 32), 0, st, p, n_cta, (int)RG);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "tree_merge_kernel launch");
    count_launches();
  }
  return HALO_OK;
}

template <typename T, int D, bool PAIR>
static int dispatch(int rows, const Params& p, int n_cta, cudaStream_t st) {
  switch (rows) {
    case 16: return launch<T, D, 16, PAIR>(p, n_cta, st);
    case 32: return launch<T, D, 32, PAIR>(p, n_cta, st);
    case 64: return launch<T, D, 64, PAIR>(p, n_cta, st);
    case 128: return launch<T, D, 128, PAIR>(p, n_cta, st);
    default: return launch<T, D, 256, PAIR>(p, n_cta, st);
  }
}

static int run(const halo_page_pool_t* pool, const halo_tree_problem_t* pb, void* workspace,
               int64_t workspace_bytes, halo_stream_t stream) {
  int rc = check(pool, pb);
  if (rc != HALO_OK) return rc;
  if (pb->R == 0 || pb->T == 0 || pb->max_nodes == 0) return HALO_OK;
  if (!pool->k || !pool->v || !pb->q || !pb->out || !pb->context_lens || !pb->cu_nodes ||
      !pb->mask || (pb->max_blocks > 0 && !pb->block_tables))
    return fail(HALO_ERR_INVALID_ARG, "NULL pointer");
  if (pb->out_dtype != HALO_DTYPE_F32 && pb->out_dtype != pool->dtype)
    return fail(HALO_ERR_UNSUPPORTED, "out dtype must be fp32 or the pool's dtype");
  // the stride of a dimension of one is never used
  const bool many_p = pool->n_pages > 1, many_h = pool->H_kv > 1;
  if (!rows16(pool->k, many_p ? pool->k_stride_p : 0, many_h ? pool->k_stride_h : 0,
              pool->k_stride_t, 2) ||
      !rows16(pool->v, many_p ? pool->v_stride_p : 0, many_h ? pool->v_stride_h : 0,
              pool->v_stride_t, 2) ||
      pool->k_stride_t <= 0 || pool->v_stride_t <= 0 ||
      (many_h && (pool->k_stride_h <= 0 || pool->v_stride_h <= 0)) ||
      (many_p && (pool->k_stride_p <= 0 || pool->v_stride_p <= 0)))
    return fail(HALO_ERR_MISALIGNED, "page rows must be 16-byte aligned, strides positive");
  if (!rows16(pb->q, pb->T > 1 ? pb->q_stride_t : 0, pb->H > 1 ? pb->q_stride_h : 0, 0, 2))
    return fail(HALO_ERR_MISALIGNED, "q rows must be 16-byte aligned");
  if (!rows16(pb->out, pb->T > 1 ? pb->out_stride_t : 0, pb->H > 1 ? pb->out_stride_h : 0, 0,
              pb->out_dtype == HALO_DTYPE_F32 ? 4 : 2))
    return fail(HALO_ERR_MISALIGNED, "out rows must be 16-byte aligned");
  if (rows_overlap(pb->T, pb->out_stride_t, pb->H, pb->out_stride_h, pool->D))
    return fail(HALO_ERR_INVALID_ARG, "out rows overlap (strides %lld %lld)",
                (long long)pb->out_stride_t, (long long)pb->out_stride_h);
  const int64_t need = ws_bytes(pool, pb);
  if (!workspace || workspace_bytes < need)
    return fail(HALO_ERR_WORKSPACE, "tree workspace has %lld bytes, needs %lld",
                (long long)(workspace ? workspace_bytes : 0), (long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) & 255)
    return fail(HALO_ERR_MISALIGNED, "tree workspace must be 256-byte aligned");

  Params p{};
  p.box = 8;
  while (p.box < kBN && pool->page_size % (2 * p.box) == 0) p.box *= 2;
  const int rows = group_rows(pool, pb);
  // Copies of 8 rows take both column blocks of 128 columns; groups of 64 rows,
  // whose one producer warp is the busiest, also halve copies of 16 rows for
  // that.  8 requests on 32768 positions, 32 / 8 heads of 128, us without and
  // with pairs on pages of 8, 16, 24, 48 and 64:
  //   16 nodes   327 212   242 217   336 230   253 233   204 236
  //    4 nodes   217 176   173 183   199 173   174 176   176 176
  // 4 requests of 64 nodes on 65535 positions: 456 434 and 516 444 on pages of 8
  // and 24, within 1 % on others.
  const bool pair = pool->D == 128 && (p.box == 8 || (p.box == 16 && rows == 64));
  if (pair) p.box = 8;
  rc = encode_pool(pool, pool->k, pool->k_stride_p, pool->k_stride_h, pool->k_stride_t, p.box,
                   pair, &p.kmap);
  if (rc != HALO_OK) return rc;
  rc = encode_pool(pool, pool->v, pool->v_stride_p, pool->v_stride_h, pool->v_stride_t, p.box,
                   pair, &p.vmap);
  if (rc != HALO_OK) return rc;
  p.q = static_cast<const char*>(pb->q);
  p.q_st = pb->q_stride_t;
  p.q_sh = pb->q_stride_h;
  p.v = static_cast<const char*>(pool->v);
  p.v_sp = pool->v_stride_p;
  p.v_sh = pool->v_stride_h;
  p.v_st = pool->v_stride_t;
  p.table = pb->block_tables;
  p.table_stride = pb->table_stride;
  p.ctx = pb->context_lens;
  p.cu = pb->cu_nodes;
  p.starts = pb->node_starts ? pb->node_starts : pb->cu_nodes;
  p.mask = pb->mask;
  p.mask_stride = pb->mask_stride;
  p.out = static_cast<char*>(pb->out);
  p.out_st = pb->out_stride_t;
  p.out_sh = pb->out_stride_h;
  p.scale_log2 = pb->scale * kLog2e;
  p.headroom = raw_headroom(p.scale_log2);
  p.out_f32 = pb->out_dtype == HALO_DTYPE_F32;
  p.R = pb->R;
  p.T = pb->T;
  p.H = pb->H;
  p.H_kv = pool->H_kv;
  p.G = pb->H / pool->H_kv;
  p.max_nodes = pb->max_nodes;
  p.max_blocks = pb->max_blocks;
  p.n_pages = pool->n_pages;
  p.page = pool->page_size;
  const int n_cta = device_sms();
  char* ws = static_cast<char*>(workspace);
  p.desc = reinterpret_cast<Desc*>(ws);
  p.part = reinterpret_cast<float*>(ws + desc_bytes(n_cta));
  p.lse = pb->lse ? pb->lse
                  : reinterpret_cast<float*>(ws + desc_bytes(n_cta) + part_bytes(pool, pb, n_cta));
  p.err = device_error_ptr();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto typed = [&](auto tag) {
    using T = decltype(tag);
    if (pool->D == 64) return dispatch<T, 64, false>(rows, p, n_cta, st);
    return pair ? dispatch<T, 128, true>(rows, p, n_cta, st)
                : dispatch<T, 128, false>(rows, p, n_cta, st);
  };
  return pool->dtype == HALO_DTYPE_BF16 ? typed(__nv_bfloat16{}) : typed(__half{});
}

}  // namespace tree
}  // namespace halo

using namespace halo;

extern "C" int64_t halo_tree_workspace_bytes(const halo_page_pool_t* pool,
                                             const halo_tree_problem_t* pb) {
  const int rc = tree::check(pool, pb);
  if (rc != HALO_OK) return rc;
  return pb->R == 0 || pb->T == 0 || pb->max_nodes == 0 ? 0 : tree::ws_bytes(pool, pb);
}

extern "C" int32_t halo_tree_attention(const halo_page_pool_t* pool, const halo_tree_problem_t* pb,
                                       void* workspace, int64_t workspace_bytes,
                                       halo_stream_t stream) {
  return tree::run(pool, pb, workspace, workspace_bytes, stream);
}
