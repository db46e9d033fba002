// mvb_paged_prefill_fp8: causal attention of a batch of prefill chunks over an
// 8-bit paged cache (codes with a scale per (block, KV head)); the chunk's own
// tokens are in the cache before the call.  Query token t of a chunk with c
// cached tokens attends positions [0, c + t].
//
// Rows.  The rows of one KV head are (token, head of its group) pairs,
// token-major, so the query heads that share keys share a tile.  A CTA holds
// two tiles of 128 rows and walks the keys 128 at a time up to its last row's
// limit:   S = Q K_codes^T,   P = exp2(S c_g - m),   O += P V.
//
// Roles (13 warps):
//   * warps 0-3 and 4-7: the softmax of row tile 0 and 1, one row per thread.
//     They read S from tensor memory twice (maximum, then exponentials), write
//     P as f16 over it, and rescale O in tensor memory only when a row's
//     maximum has risen by more than 8 (in powers of two; P <= 2^8 then);
//   * warps 8-11: the loaders.  They read codes through the block table one
//     tile ahead, turn them into f16 (exact) and store K and V tiles in the
//     128-byte swizzled layout that the tensor core reads, 2 stages each;
//   * warp 12: issues the tensor-core products (tcgen05.mma, 128 x 128 and
//     128 x D per tile): S of one row tile runs while the other is in its softmax.
//
// Scales.  A block's key scale is one factor of 16 columns of S (a group), so it
// joins the softmax scale in the exponent's multiply-add at no cost.  Values
// enter as code * 2^e, e the exponent of (the power of two in) the block's scale
// over a reference R of the tile's largest; the product is exact in f16 for
// scales from 2^-15 R to 2^7 R, and R (and O with it) moves when a scale passes
// 2^7 R.  The rest of a scale that is no power of two multiplies P.
//
// The query enters as f16, each row times a power of two that brings its
// largest element into [1, 2) (as in the decode kernel, fp8_decode.cu).
//
// A NaN among the values must not reach rows that do not attend it (0 * NaN):
// the loaders replace NaN codes by 0 and leave a bit per (key, column); a row
// that attends the key gets NaN in that column at the end.
//
// Bound: 16384 exponentials per 128 x 128 tile at 16 per cycle and SM for
// head_dim 64, the tensor core for head_dim 128.
//
// Every wait is bounded (kWaitSpinLimit); one that runs out sets
// MVB_DEV_TIMEOUT, tells the other roles to leave, and the CTA waits (bounded)
// for its products in flight before it frees its tensor memory.
#include "fp8_common.cuh"

namespace mvb {

struct Fp8PrefillArgs {
  const void* q;
  int64_t q_s0, q_s1;
  const uint8_t* kc;
  const uint8_t* vc;
  const float2* scale;  // [num_blocks, KH] (key, value)
  const int64_t* bt;
  int64_t bt_rows, bt_s0;
  int max_blocks;
  const int64_t* seq_rows;
  const int64_t* cached;
  const int64_t* qlen;
  int n, total_q;
  void* out;
  int64_t o_s0, o_s1;
  int num_heads, num_kv_heads, G, block_shift, num_blocks;
  float scale_log2;
  int* err;
};

namespace {

constexpr int kFp8PrefillMaxChunks = 4096;
constexpr int kTileRows = 128;               // rows of one row tile (tensor-core M)
constexpr int kCtaRows = 2 * kTileRows;      // (token, head) rows of one CTA
constexpr int kKeys = 128;                   // keys per step
constexpr int kGroups = kKeys / 16;          // 16-key groups: each lies in one block
constexpr int kThreads = 13 * 32;
constexpr int kInfos = 4;                    // steps whose side information is kept
constexpr int kTmemCols = 512;

// Side information of one step, written by the loaders.
struct StepInfo {
  float ks[kGroups];  // key scales
  float vf[kGroups];  // value scale over its power of two, in [1, 2)
  float r;            // reference R of the values (O is in units of it)
  float rf;           // the previous step's R over this one's
  int bad;            // bit g: the group's block id is invalid, its keys are left out
  int nan[4];         // per loader warp: the step's values hold NaN
};

template <int D> struct Geo {
  static constexpr int QBYTES = kTileRows * D * 2, KBYTES = kKeys * D * 2;
  static constexpr int NMASK = kInfos * kKeys * (D / 16) * 2;  // a bit per (key, column)
  static constexpr int Q = 0, K = 2 * QBYTES, V = K + 2 * KBYTES, MASK = V + 2 * KBYTES;
  static constexpr int INFO = MASK + NMASK, BARS = INFO + kInfos * (int)sizeof(StepInfo);
  static constexpr int BYTES = BARS + 128 + 1024;  // + alignment
  static constexpr int S_COL = 0, O_COL = 256;     // tensor-memory columns: S 2 x 128, O 2 x D
};

// Barriers (indices).
enum { kQ = 0, kKFull = 1, kKEmpty = 3, kVFull = 5, kVEmpty = 7, kSFull = 9, kPReady = 11, kPvDone = 13, kNumBars = 15 };

// ---- tensor memory and tcgen05 ----------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t smem_dst) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "n"(kTmemCols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "n"(kTmemCols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 32 consecutive columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Shared-memory operand in the 128-byte swizzle: `lead` and `stride` in bytes.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 |
         (uint64_t)((stride >> 4) & 0x3fff) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Instruction word: f16 operands, f32 result, M = 128, B transposed (N contiguous) or not.
constexpr uint32_t mma_word(int n, bool b_mn_major) {
  return 1u << 4 | (b_mn_major ? 1u << 16 : 0u) | (uint32_t)(n / 8) << 17 | (uint32_t)(kTileRows / 16) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t word, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(word), "r"((int)add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t word, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(word),
      "r"((int)add)
      : "memory");
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, __half2 f) {
  const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&a), f);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Byte offset of 16-byte chunk `c` of a row's 64-column panel in a swizzled tile of 128 rows.
__device__ __forceinline__ uint32_t swz(int row, int panel, int c) {
  return (uint32_t)(panel * (kKeys * 128) + row * 128 + ((c ^ (row & 7)) << 4));
}
// The power of two in a positive scale (0 for 0 and for scales below 2^-126).
__device__ __forceinline__ float pow2_of(float s) { return __uint_as_float(__float_as_uint(s) & 0x7f800000u); }

// Waits of all roles: bounded, and given up when another role has given up.
struct Waiter {
  uint32_t bars;
  volatile int* stop;
  int* err;
  __device__ __forceinline__ uint32_t bar(int i) const { return bars + 8 * i; }
  __device__ __forceinline__ bool operator()(int i, int parity) const {
    for (int n = 0; n < kWaitSpinLimit; ++n) {
      if (mbar_try_wait(bar(i), (uint32_t)parity)) return true;
      if ((n & 63) == 63 && *stop) return false;
    }
    *stop = 1;
    atomicOr(err, MVB_DEV_TIMEOUT);
    return false;
  }
  // All lanes of a warp, which stay together whatever each of them saw.
  __device__ __forceinline__ bool warp(int i, int parity) const {
    return __all_sync(0xffffffffu, (*this)(i, parity)) != 0;
  }
};

// Columns [0, 32) of a chunk of S as P (f16 pairs), their sum added to l.
// EDGE: the step holds keys that some row does not attend (lim: the row's keys in
// this chunk; bad: bits of the chunk's two groups that are left out).
template <bool EDGE>
__device__ __forceinline__ float chunk_max(const uint32_t (&s)[32], float mx, const float* c, int lim, int bad) {
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = __uint_as_float(s[16 * g + i]);
      if (EDGE && (16 * g + i >= lim || (bad >> g & 1))) v = -INFINITY;
      x[i & 3] = fmaxf(x[i & 3], v);
    }
    mx = fmaxf(mx, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * c[g]);
  }
  return mx;
}
template <bool EDGE>
__device__ __forceinline__ void chunk_exp(const uint32_t (&s)[32], uint32_t (&p)[16], float m, const float* c,
                                          const float* vf, int lim, int bad, float (&l)[2]) {
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    float e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float y = fmaf(__uint_as_float(s[16 * g + i]), c[g], -m);
      if (EDGE && (16 * g + i >= lim || (bad >> g & 1))) y = -INFINITY;
      e[i] = fast_exp2(y);
      l[i & 1] += e[i];
    }
    if (vf[g] != 1.f) {  // a value scale that is no power of two
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] *= vf[g];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) p[8 * g + i] = pack_h2(e[2 * i], e[2 * i + 1]);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) fp8_prefill_kernel(const Fp8PrefillArgs a) {
  using G_ = Geo<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int s_tot[2][kThreads / 32];
  __shared__ uint32_t s_tmem;
  __shared__ int s_stop;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- row tiles and tokens of every chunk, exclusive prefixes (they lie where the stages will) ----
  int* pre = reinterpret_cast<int*>(smem + G_::K);  // [n + 1]
  int* qpre = pre + a.n + 1;                        // [n + 1]
  {
    const int per = (a.n + kThreads - 1) / kThreads;
    const int i0 = min(a.n, tid * per), i1 = min(a.n, i0 + per);
    int mt = 0, mq = 0;
    for (int i = i0; i < i1; ++i) {
      const int ql = (int)min((int64_t)a.total_q + 1, max((int64_t)0, __ldg(a.qlen + i)));
      pre[i] = (int)(((int64_t)ql * a.G + kCtaRows - 1) / kCtaRows);
      qpre[i] = ql;
      mt += pre[i];
      mq = min(mq + ql, a.total_q + 1);
    }
    int it = mt, iq = mq;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int vt = __shfl_up_sync(0xffffffffu, it, o), vq = __shfl_up_sync(0xffffffffu, iq, o);
      if (lane >= o) {
        it += vt;
        iq = min(iq + vq, a.total_q + 1);
      }
    }
    if (lane == 31) {
      s_tot[0][warp] = it;
      s_tot[1][warp] = iq;
    }
    __syncthreads();
    int rt = 0, rq = 0, Tt = 0, Tq = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w == warp) {
        rt = Tt;
        rq = Tq;
      }
      Tt += s_tot[0][w];
      Tq = min(Tq + s_tot[1][w], a.total_q + 1);
    }
    rt += it - mt;
    rq = min(rq + iq - mq, a.total_q + 1);
    for (int i = i0; i < i1; ++i) {
      const int t = pre[i], q = qpre[i];
      pre[i] = rt;
      qpre[i] = rq;
      rt += t;
      rq = min(rq + q, a.total_q + 1);
    }
    if (tid == 0) {
      pre[a.n] = Tt;
      qpre[a.n] = Tq;
    }
    __syncthreads();
  }
  if (qpre[a.n] > a.total_q) {  // the chunks hold more tokens than query has rows: refuse
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) atomicOr(a.err, MVB_DEV_BLOCK_ID);
    return;
  }
  const int x = pre[a.n] - 1 - (int)blockIdx.x;  // a chunk's last rows first: they attend most keys
  if (x < 0) return;
  int lo = 0, hi = a.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  const int kvh = blockIdx.y, h0 = kvh * a.G;
  const int q0 = qpre[lo], ql = qpre[lo + 1] - q0, rows = ql * a.G;
  const int row0 = (x - pre[lo]) * kCtaRows;  // the CTA's first row in the chunk
  const int nrows = min(kCtaRows, rows - row0);
  const int64_t srow = __ldg(a.seq_rows + lo), cached = __ldg(a.cached + lo);
  T* const out = static_cast<T*>(a.out);
  if (cached < 0 || srow < 0 || srow >= a.bt_rows ||
      (cached + ql + (1 << a.block_shift) - 1) >> a.block_shift > a.max_blocks) {
    // a table too short for the chunk (or a bad row): zeros, and the flag
    if (tid == 0) atomicOr(a.err, MVB_DEV_TABLE_SHORT);
    for (int e = tid; e < nrows * D; e += kThreads) {
      const int r = row0 + e / D;
      out[(int64_t)(q0 + r / a.G) * a.o_s0 + (int64_t)(h0 + r % a.G) * a.o_s1 + e % D] = from_f32<T>(0.f);
    }
    return;
  }
  const int kv_end = (int)cached + (row0 + nrows - 1) / a.G + 1;  // positions the CTA's last row attends
  const int steps = (kv_end + kKeys - 1) / kKeys;
  const int tiles = nrows > kTileRows ? 2 : 1;

  Waiter wait;
  wait.bars = smem_u32(smem + G_::BARS);
  wait.stop = &s_stop;
  wait.err = a.err;
  StepInfo* infos = reinterpret_cast<StepInfo*>(smem + G_::INFO);
  uint16_t* masks = reinterpret_cast<uint16_t*>(smem + G_::MASK);  // [kInfos][kKeys][D / 16]
  if (warp == 12) tmem_alloc(smem_u32(&s_tmem));
  if (tid == 0) {
    s_stop = 0;
    mbar_init(wait.bar(kQ), 4 * tiles);
    for (int i = 0; i < 2; ++i) {
      mbar_init(wait.bar(kKFull + i), 4);
      mbar_init(wait.bar(kVFull + i), 4);
      mbar_init(wait.bar(kKEmpty + i), 1);
      mbar_init(wait.bar(kVEmpty + i), 1);
      mbar_init(wait.bar(kSFull + i), 1);
      mbar_init(wait.bar(kPReady + i), 4);
      mbar_init(wait.bar(kPvDone + i), 1);
    }
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  if (warp < 8) {
    // ================================ softmax =================================
    const int tile = warp >> 2, r = row0 + tile * kTileRows + (warp & 3) * 32 + lane;
    if (tile < tiles) {
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t s_at = tmem + lanes + G_::S_COL + tile * kKeys, o_at = tmem + lanes + G_::O_COL + tile * D;
      const bool live = r < rows;
      const int tok = live ? r / a.G : 0, head = live ? r - tok * a.G : 0;
      const int lim = live ? (int)cached + tok + 1 : kv_end;  // rows past the chunk are zeros that attend all
      float qs;
      {
        const uint4* qp = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (int64_t)(q0 + tok) * a.q_s0 +
                                                         (int64_t)(h0 + head) * a.q_s1);
        uint4 raw[D / 8];
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          raw[i] = live ? __ldg(qp + i) : make_uint4(0, 0, 0, 0);
          const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float y = fabsf(to_f32<T>(e[k]));
            amax = fmaxf(amax, y < INFINITY ? y : 0.f);
          }
        }
        const int e2 = min(max((int)(__float_as_uint(amax) >> 23), 2), 252);
        // the softmax scale's sign goes with the query: the maximum below is over S times a positive factor
        const float down = copysignf(__uint_as_float((uint32_t)(254 - e2) << 23), a.scale_log2);
        qs = fabsf(a.scale_log2) * __uint_as_float((uint32_t)e2 << 23);
        uint8_t* qd = smem + G_::Q + tile * G_::QBYTES;
        const int qr = (warp & 3) * 32 + lane;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const T* e = reinterpret_cast<const T*>(&raw[i]);
          uint4 w;
          w.x = pack_h2(to_f32<T>(e[0]) * down, to_f32<T>(e[1]) * down);
          w.y = pack_h2(to_f32<T>(e[2]) * down, to_f32<T>(e[3]) * down);
          w.z = pack_h2(to_f32<T>(e[4]) * down, to_f32<T>(e[5]) * down);
          w.w = pack_h2(to_f32<T>(e[6]) * down, to_f32<T>(e[7]) * down);
          *reinterpret_cast<uint4*>(qd + swz(qr, i / 8, i % 8)) = w;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(wait.bar(kQ));
      }
      float m = -INFINITY, l[2] = {0.f, 0.f};
      uint32_t nanbits[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) nanbits[i] = 0u;
      auto take_nan = [&](int j) {  // columns of step j's values that are NaN for this row
        const StepInfo& f = infos[j % kInfos];
        if (!(f.nan[0] | f.nan[1] | f.nan[2] | f.nan[3])) return;
        const int n = min(kKeys, lim - j * kKeys);
        for (int k = 0; k < n; ++k)
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
            nanbits[i] |= reinterpret_cast<const uint32_t*>(masks + ((j % kInfos) * kKeys + k) * (D / 16))[i];
      };
      bool ok = true;
      for (int j = 0; j < steps; ++j) {
        if (!wait.warp(kSFull + tile, j & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (j > 0) take_nan(j - 1);  // (its products are done: S of this step was issued after them)
        const StepInfo& f = infos[j % kInfos];
        const int rem = lim - j * kKeys, bad = f.bad;
        const bool edge = __any_sync(0xffffffffu, rem < kKeys) || bad != 0;
        float c[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) c[g] = qs * f.ks[g];
        uint32_t s[32];
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          tmem_ld32(s_at + 32 * h, s);
          tc_wait_ld();
          mx = edge ? chunk_max<true>(s, mx, c + 2 * h, rem - 32 * h, bad >> (2 * h))
                    : chunk_max<false>(s, mx, c + 2 * h, 0, 0);
        }
        const bool jump = mx > m + 8.f;
        const float rf = f.rf;
        if (__any_sync(0xffffffffu, jump) || rf != 1.f) {
          const float mn = jump ? mx : m, al = jump ? fast_exp2(m - mn) : 1.f;
          m = mn;
          l[0] *= al;
          l[1] *= al;
          if (j > 0) {
            const float fac = al * rf;
#pragma unroll
            for (int h = 0; h < D / 32; ++h) {
              uint32_t o[32];
              tmem_ld32(o_at + 32 * h, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fac);
              tmem_st32(o_at + 32 * h, o);
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t p[16];
          tmem_ld32(s_at + 32 * h, s);
          tc_wait_ld();
          if (edge)
            chunk_exp<true>(s, p, m, c + 2 * h, f.vf + 2 * h, rem - 32 * h, bad >> (2 * h), l);
          else
            chunk_exp<false>(s, p, m, c + 2 * h, f.vf + 2 * h, 0, 0, l);
          tmem_st16(s_at + 16 * h, p);  // over columns of S that have been read
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(wait.bar(kPReady + tile));
      }
      if (ok && wait.warp(kPvDone + tile, (steps - 1) & 1)) {
        tc_fence_after();
        take_nan(steps - 1);
        const float sum = l[0] + l[1];
        const float inv = sum == 0.f ? 0.f : infos[(steps - 1) % kInfos].r / sum;
        T* op = out + (int64_t)(q0 + tok) * a.o_s0 + (int64_t)(h0 + head) * a.o_s1;
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
          uint32_t o[32];
          tmem_ld32(o_at + 32 * h, o);
          tc_wait_ld();
          if (!live) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 w;
            T* e = reinterpret_cast<T*>(&w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float v = __uint_as_float(o[8 * i + k]) * inv;
              e[k] = from_f32<T>((nanbits[h] >> (8 * i + k)) & 1 ? __uint_as_float(0x7fffffffu) : v);
            }
            *reinterpret_cast<uint4*>(op + 32 * h + 8 * i) = w;
          }
        }
      }
    }
  } else if (warp < 12) {
    // ================================ loaders =================================
    constexpr int CH = D / 16, N = kKeys * CH / 128;  // 16-code chunks per row, chunks per thread and tile
    const int lt = tid - 256, lw = warp - 8;
    const int64_t* bt = a.bt + srow * a.bt_s0;
    const int BSm = (1 << a.block_shift) - 1, grp = lane & (kGroups - 1);
    // lane g (and g + 8, ..): where 16-key group g of a step lies: (block, KV head) row, -1 behind the last key or bad
    auto find = [&](int j, bool& bad) {
      const int p = j * kKeys + 16 * grp;
      bad = false;
      if (p >= kv_end) return -1;
      const int64_t b = __ldg(bt + (p >> a.block_shift));
      bad = b < 0 || b >= a.num_blocks;
      return bad ? -1 : (int)(b * a.num_kv_heads + kvh);
    };
    uint4 kr[N], vr[N];
    auto fetch = [&](uint4 (&d)[N], const uint8_t* base, int j, int row) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int key = lt / CH + i * (128 / CH), p = j * kKeys + key;
        const int rw = __shfl_sync(0xffffffffu, row, key >> 4);
        d[i] = make_uint4(0, 0, 0, 0);
        if (rw >= 0 && p < kv_end)
          d[i] = __ldg(reinterpret_cast<const uint4*>(base + (((int64_t)rw << a.block_shift) + (p & BSm)) * D) +
                       lt % CH);
      }
    };
    bool bad, bad_n = false;
    int row = find(0, bad), row_n = -1;
    float2 sc = row >= 0 ? __ldg(a.scale + row) : make_float2(0.f, 0.f);
    fetch(kr, a.kc, 0, row);
    fetch(vr, a.vc, 0, row);
    if (steps > 1) row_n = find(1, bad_n);
    float R = 1.f;
    for (int j = 0; j < steps; ++j) {
      const int st = j & 1;
      float2 sc_n = row_n >= 0 ? __ldg(a.scale + row_n) : make_float2(0.f, 0.f);
      // the values' reference, and each group's factor
      float vp = pow2_of(sc.y), top = vp;
#pragma unroll
      for (int o = 1; o < kGroups; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float rf = 1.f;
      if (j == 0)
        R = top > 0.f ? top : 1.f;
      else if (top > 128.f * R) {
        rf = R / top;
        R = top;
      }
      const float vscale = vp / R;
      StepInfo& f = infos[j % kInfos];
      const uint32_t badmask = __ballot_sync(0xffffffffu, bad) & ((1u << kGroups) - 1);
      if (lw == 0) {
        if (lane < kGroups) {
          f.ks[lane] = sc.x;
          f.vf[lane] = vp > 0.f ? sc.y / vp : 1.f;
        }
        if (lane == 0) {
          f.r = R;
          f.rf = rf;
          f.bad = (int)badmask;
          if (badmask) atomicOr(a.err, MVB_DEV_BLOCK_ID);
        }
      }
      if (j >= 2 && !wait.warp(kKEmpty + st, (j / 2 - 1) & 1)) break;
      uint8_t* kd = smem + G_::K + st * G_::KBYTES;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int key = lt / CH + i * (128 / CH), ch = lt % CH;
        uint4 w0, w1;
        e4m3x4_to_f16(kr[i].x, w0.x, w0.y);
        e4m3x4_to_f16(kr[i].y, w0.z, w0.w);
        e4m3x4_to_f16(kr[i].z, w1.x, w1.y);
        e4m3x4_to_f16(kr[i].w, w1.z, w1.w);
        *reinterpret_cast<uint4*>(kd + swz(key, ch / 4, 2 * (ch % 4))) = w0;
        *reinterpret_cast<uint4*>(kd + swz(key, ch / 4, 2 * (ch % 4) + 1)) = w1;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(wait.bar(kKFull + st));
      if (j + 1 < steps) fetch(kr, a.kc, j + 1, row_n);

      if (j >= 2 && !wait.warp(kVEmpty + st, (j / 2 - 1) & 1)) break;
      uint8_t* vd = smem + G_::V + st * G_::KBYTES;
      bool any_nan = false;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int key = lt / CH + i * (128 / CH), ch = lt % CH;
        uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w}, nan16 = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t n = ((w[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // bytes 0x7f and 0xff: NaN
          if (n) {
            w[k] &= ~((n >> 7) * 0xffu);
            nan16 |= ((n >> 7 & 1) | (n >> 14 & 2) | (n >> 21 & 4) | (n >> 28 & 8)) << (4 * k);
          }
        }
        any_nan |= nan16 != 0;
        masks[((j % kInfos) * kKeys + key) * CH + ch] = (uint16_t)nan16;
        const __half2 vs = __float2half2_rn(__shfl_sync(0xffffffffu, vscale, key >> 4));
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          e4m3x4_to_f16(w[k], h[2 * k], h[2 * k + 1]);
          h[2 * k] = mul_h2(h[2 * k], vs);
          h[2 * k + 1] = mul_h2(h[2 * k + 1], vs);
        }
        *reinterpret_cast<uint4*>(vd + swz(key, ch / 4, 2 * (ch % 4))) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(vd + swz(key, ch / 4, 2 * (ch % 4) + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
      any_nan = __any_sync(0xffffffffu, any_nan);
      if (lane == 0) f.nan[lw] = any_nan;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(wait.bar(kVFull + st));
      if (j + 1 < steps) fetch(vr, a.vc, j + 1, row_n);
      row = row_n;
      bad = bad_n;
      sc = sc_n;
      row_n = -1;
      bad_n = false;
      if (j + 2 < steps) row_n = find(j + 2, bad_n);
    }
  } else if (lane == 0) {
    // ========================= tensor-core products ===========================
    const uint32_t base = smem_u32(smem);
    constexpr uint32_t SW = mma_word(kKeys, false), PW = mma_word(D, true);
    auto scores = [&](int i, int st) {  // S_i = Q_i K^T: 16 columns (32 bytes of a panel's row) a step
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (uint32_t)((k / 4) * (kKeys * 128) + (k % 4) * 32);
        mma_ss(tmem + G_::S_COL + i * kKeys, smem_desc(base + G_::Q + i * G_::QBYTES + off, 16, 1024),
               smem_desc(base + G_::K + st * G_::KBYTES + off, 16, 1024), SW, k > 0);
      }
      tc_commit(wait.bar(kSFull + i));
    };
    auto values = [&](int i, int st, bool add) {  // O_i += P_i V: 16 keys (2 KB of a panel) a step
#pragma unroll
      for (int k = 0; k < kKeys / 16; ++k)
        mma_ts(tmem + G_::O_COL + i * D, tmem + G_::S_COL + i * kKeys + 8 * k,
               smem_desc(base + G_::V + st * G_::KBYTES + k * 2048, kKeys * 128, 1024), PW, add || k > 0);
      tc_commit(wait.bar(kPvDone + i));
    };
    bool ok = wait(kQ, 0) && wait(kKFull, 0);
    if (ok) {
      tc_fence_after();
      for (int i = 0; i < tiles; ++i) scores(i, 0);
      tc_commit(wait.bar(kKEmpty));
    }
    for (int j = 0; ok && j < steps; ++j) {
      const int st = j & 1, sn = st ^ 1;
      for (int i = 0; ok && i < tiles; ++i) {
        ok = (i > 0 || wait(kVFull + st, (j / 2) & 1)) && wait(kPReady + i, j & 1);
        if (!ok) break;
        tc_fence_after();
        values(i, st, j > 0);
        if (i == tiles - 1) tc_commit(wait.bar(kVEmpty + st));
        if (j + 1 < steps) {
          // S of the next step overwrites P: the products that read it come first
          ok = (i > 0 || wait(kKFull + sn, ((j + 1) / 2) & 1)) && wait(kPvDone + i, j & 1);
          if (!ok) break;
          tc_fence_after();
          scores(i, sn);
          if (i == tiles - 1) tc_commit(wait.bar(kKEmpty + sn));
        }
      }
    }
    if (!ok) {
      // given up: wait for whatever was issued before the tensor memory goes (the last commit's barrier has
      // one arrival per phase, so its phase is unknown here: use one that nothing else waits on any more)
      mbar_init(wait.bar(kNumBars), 1);
      fence_mbar_init();
      tc_commit(wait.bar(kNumBars));
      mbar_wait_bounded(wait.bar(kNumBars), 0);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_free(tmem);
}

template <typename T, int D>
int launch_prefill_fp8(const Fp8PrefillArgs& a, cudaStream_t stream) {
  auto kern = fp8_prefill_kernel<T, D>;
  static_assert(2 * (kFp8PrefillMaxChunks + 1) * 4 <= 4 * Geo<D>::KBYTES, "the prefixes fit the stages");
  static_assert(Geo<D>::BYTES <= 227 * 1024 - 512, "shared memory of one CTA");
  if (ensure_kernel_attrs(kern, Geo<D>::BYTES) != cudaSuccess) return MVB_ERR_CUDA;
  const int64_t tiles = ((int64_t)a.total_q * a.G + kCtaRows - 1) / kCtaRows + a.n;
  return launch_pdl(kern, dim3((unsigned)tiles, a.num_kv_heads), dim3(kThreads), Geo<D>::BYTES, stream, a) ==
                 cudaSuccess
             ? MVB_OK
             : MVB_ERR_CUDA;
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int mvb_paged_prefill_fp8(const void* query, int64_t q_stride_tok, int64_t q_stride_head,
                                     const void* key_cache, const void* value_cache, const float* kv_scale,
                                     const int64_t* block_table, int64_t block_table_rows,
                                     int64_t block_table_stride, int32_t max_blocks_per_seq, const int64_t* seq_rows,
                                     const int64_t* cached_len, const int64_t* query_len, int32_t num_chunks,
                                     int32_t total_q, void* out, int64_t out_stride_tok, int64_t out_stride_head,
                                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                     int32_t num_blocks, float scale, int32_t dtype, int32_t* error_flags,
                                     void* stream) {
  mvb::NvtxRange nvtx_range("mvb_paged_prefill_fp8");
  if (dtype != MVB_DTYPE_F16 && dtype != MVB_DTYPE_BF16) return MVB_ERR_DTYPE;
  if (head_dim != 64 && head_dim != 128) return MVB_ERR_HEAD_DIM;
  if (block_size < kFp8MinBlock || block_size > kFp8MaxBlock || (block_size & (block_size - 1)) != 0)
    return MVB_ERR_BLOCK_SIZE;
  if (num_chunks < 0 || num_chunks > kFp8PrefillMaxChunks || total_q < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_kv_heads > 65535 || num_blocks <= 0 || max_blocks_per_seq < 0 || block_table_rows < 0)
    return MVB_ERR_INVALID_ARG;
  if (num_heads % num_kv_heads != 0) return MVB_ERR_HEADS;
  const int G = num_heads / num_kv_heads;
  // rows of a KV head, positions of a sequence and (block, KV head) numbers are 32-bit
  if ((int64_t)total_q * G >= ((int64_t)1 << 30) || (int64_t)max_blocks_per_seq * block_size >= ((int64_t)1 << 30) ||
      (int64_t)num_blocks * num_kv_heads >= ((int64_t)1 << 31))
    return MVB_ERR_INVALID_ARG;
  if (num_chunks == 0 || total_q == 0) return MVB_OK;
  if (!query || !key_cache || !value_cache || !kv_scale || !block_table || !seq_rows || !cached_len || !query_len ||
      !out || !error_flags)
    return MVB_ERR_INVALID_ARG;
  if (max_blocks_per_seq > 0 && block_table_stride < max_blocks_per_seq) return MVB_ERR_INVALID_ARG;
  auto al = [](const void* p, int64_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!al(query, 16) || q_stride_tok % 8 || q_stride_head % 8 || !al(out, 16) || out_stride_tok % 8 ||
      out_stride_head % 8 || !al(key_cache, 16) || !al(value_cache, 16) || !al(kv_scale, 8))
    return MVB_ERR_ALIGNMENT;
  Fp8PrefillArgs a;
  a.q = query;
  a.q_s0 = q_stride_tok;
  a.q_s1 = q_stride_head;
  a.kc = static_cast<const uint8_t*>(key_cache);
  a.vc = static_cast<const uint8_t*>(value_cache);
  a.scale = reinterpret_cast<const float2*>(kv_scale);
  a.bt = block_table;
  a.bt_rows = block_table_rows;
  a.bt_s0 = block_table_stride;
  a.max_blocks = max_blocks_per_seq;
  a.seq_rows = seq_rows;
  a.cached = cached_len;
  a.qlen = query_len;
  a.n = num_chunks;
  a.total_q = total_q;
  a.out = out;
  a.o_s0 = out_stride_tok;
  a.o_s1 = out_stride_head;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.G = G;
  a.block_shift = 31 - __builtin_clz(block_size);
  a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err = error_flags;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MVB_DTYPE_BF16)
    return head_dim == 64 ? launch_prefill_fp8<__nv_bfloat16, 64>(a, s) : launch_prefill_fp8<__nv_bfloat16, 128>(a, s);
  return head_dim == 64 ? launch_prefill_fp8<__half, 64>(a, s) : launch_prefill_fp8<__half, 128>(a, s);
}
