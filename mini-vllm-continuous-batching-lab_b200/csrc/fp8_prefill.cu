// mvb_paged_prefill_fp8: causal attention of a batch of prefill chunks over an
// 8-bit paged cache (codes with a scale per (block, KV head)); the chunk's own
// tokens are in the cache before the call.  Query token t of a chunk with c
// cached tokens attends positions [0, c + t].
//
// Rows.  The rows of one KV head are (token, head of its group) pairs,
// token-major, so the query heads that share keys share a tile.  A CTA holds
// two tiles of 128 rows and walks the keys 64 at a time up to its last row's limit:
//   S = Q K_codes^T,   P = exp2(S c_g - m),   O += P V.
//
// Roles (warpgroups; registers move from the last ones to the softmax):
//   * two of softmax, one per row tile, one row per thread.  A step takes its
//     exponentials against a maximum of earlier steps and reads S once.  P may then
//     exceed 1; only when 16 of them add up to more than 2^14 (so that f16 never
//     overflows) is the maximum taken anew, O rescaled in tensor memory and the
//     step repeated, once.  P goes to tensor memory as f16, over S;
//   * one that loads K and one that loads V.  They copy codes through the block
//     table one step ahead into shared memory (cp.async; block ids and scales are
//     read eight to sixteen steps ahead), turn them into f16 (exact) and store tiles
//     in the 128-byte swizzled layout that the tensor core reads, three stages each;
//   * one warp per row tile issues its tensor-core products (tcgen05.mma, 128 x 64
//     and 128 x D per step).  A tile has two buffers of S, so the next step's scores
//     are there when its softmax comes to them, and the two tiles run independently.
//
// Scales.  A block's key scale is one factor of 16 columns of S (a group), so it
// joins the softmax scale in the exponent's multiply-add at no cost.  A value
// scale v joins the exponent too: P = p v / R, with the sum of p undone per
// group, and O is in units of R, a power of two.  R is the largest scale of the
// first step that has one above 0, and moves (O with it) when a scale passes
// 2^7 R.  The exponent takes v / R down to 2^-4, where P's f16 still has 10 bits
// for p >= 2^-10; the rest of a smaller scale goes into the f16 codes (exact to
// 2^-15 R).
//
// Few rows (fewer CTAs than SMs): several CTAs share a row tile's keys, each leaves its
// result and the log2 of its sum of exponentials in the workspace, and
// fp8_prefill_merge_kernel joins them.
//
// The query enters as f16, each row times a power of two that brings its
// largest element into [1, 2) (as in the decode kernel, fp8_decode.cu).
//
// A NaN among the values must not reach rows that do not attend it (0 * NaN):
// the loaders replace NaN codes by 0 and leave a bit per (key, column); a row
// that attends the key gets NaN in that column at the end.
//
// Bound: a step (256 rows, 64 keys) has 1024 cycles of exponentials (16 per cycle
// and SM) and, for head_dim 128, 1024 of the tensor core.  It takes about 2300: the
// scores are always there when a softmax warp looks, and its own instructions in
// turn (two such warps per scheduler) are what the step waits for; no unit is busy
// for half of the time.  Tried (8192 tokens, against 287 us then): columns read 32 or 64
// at a time: 308, 298; four row tiles of one S buffer each (16 softmax warps, each
// of which then waits for its products): 318; two warps per row, each with half of a
// step's keys and an O of its own: 284 to 290, and 20 against 17.5 us for 37 tokens;
// loaders that bring two steps at once: 296; 128 keys a step with one buffer of S:
// 278, but 939 against 834 us for head_dim 128, whose P then has to wait in registers
// for S to be read.
// Measured: 8192 tokens, 14/2 heads of 64: 275 us, 437 TFLOP/s; 4 x 2048 tokens,
// 32/8 heads of 128 after 3000 to 6144 cached: 820 us, 770 TFLOP/s.
//
// Every wait is bounded (kWaitSpinLimit), as every loop is; one that runs out sets
// MVB_DEV_TIMEOUT, tells the other roles to leave, and the CTA waits (bounded)
// for its products in flight before it frees its tensor memory.
#include <algorithm>
#include <type_traits>

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
  int splits;  // CTAs that share the keys of a row tile
  float* part; // splits > 1: [splits][total_q][num_heads][D] results, then [splits][total_q][num_heads] log2 of sums
  int* err;
};

namespace {

constexpr int kFp8PrefillMaxChunks = 4096;
constexpr int kTileRows = 128;      // rows of one row tile (tensor-core M)
constexpr int kKeys = 64;           // keys per step
constexpr int kGroups = kKeys / 16; // 16-key groups: each lies in one block
constexpr int kBatch = 32 / kGroups;  // steps whose groups the lanes of a warp hold
constexpr int kInfos = 2 * kBatch;  // steps whose side information is kept
constexpr int kStages = 3;          // of K and of V
constexpr int kNanLag = 3;          // the softmax takes a step's NaN masks this much later
constexpr int kMasks = kStages + kNanLag;  // steps whose NaN masks are kept
constexpr int kTmemCols = 512;
constexpr int kMinSteps = 2;        // of one of the CTAs that share a row tile's keys
constexpr int kMaxSplits = 16;
constexpr int kMinValueExp = -4;      // of the part of a value scale that joins the exponent

// Side information of one step, written by the loaders (nan by those of V).
struct alignas(16) StepInfo {
  // per group: the key scale; log2 of the part ve of (value scale / R) that goes into P; 2^-ve
  float4 g[kGroups];
  float r;            // reference R of the values (O is in units of it)
  float rf;           // the previous step's R over this one's
  int bad;            // bit g: the group's block id is invalid, its keys are left out
  int nan[4];         // per loader warp: its keys' values hold NaN, and their masks are written
};

constexpr int NT = 2;  // row tiles
constexpr int NB = 2;  // buffers of S (and P) per tile
constexpr int kThreads = 128 * (NT + 3), kCtaRows = NT * kTileRows;
constexpr int kLoadWarp = 4 * NT, kMmaWarp = kLoadWarp + 8;  // first warps of the roles behind the softmax

template <int D> struct Geo {
  // registers: launched with LAUNCH, moved to what each role takes
  static constexpr int LAUNCH = 96, SOFTMAX = D == 64 ? 144 : 152, LOADER = D == 64 ? 72 : 64, MMA = 48;
  static_assert(NT * SOFTMAX + 2 * LOADER + MMA <= (NT + 3) * LAUNCH, "what the block was launched with");
  static constexpr int QBYTES = kTileRows * D * 2, KBYTES = kKeys * D * 2, RAWBYTES = kKeys * D;
  static constexpr int Q = 0, K = NT * QBYTES, V = K + kStages * KBYTES, RAW = V + kStages * KBYTES;  // RAW: K, V codes
  static constexpr int MASK = RAW + 2 * RAWBYTES, NMASK = kMasks * kKeys * (D / 16) * 2;  // a bit per (key, column)
  static constexpr int INFO = MASK + NMASK, BARS = INFO + kInfos * (int)sizeof(StepInfo);
  static constexpr int BYTES = BARS + 256 + 1024;  // + alignment
  // tensor-memory columns: S (and P over its first half) NT x NB x 64, O NT x D
  static constexpr int O_COL = NT * NB * kKeys;
  static_assert(O_COL + NT * D <= kTmemCols, "tensor memory");
};

// Barriers (indices): per stage; per tile and buffer of S (so that no one's wait is ever two phases off).
enum {
  kQ = 0,
  kKFull = 1,
  kKEmpty = kKFull + kStages,
  kVFull = kKEmpty + kStages,
  kVEmpty = kVFull + kStages,
  kSFull = kVEmpty + kStages,
  kPReady = kSFull + 4,
  kPvDone = kPReady + 4,
  kGivenUp = kPvDone + 4,  // per tile, used once
  kNumBars = kGivenUp + 4
};
static_assert(kNumBars * 8 <= 256, "the barriers' place");

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
__device__ __forceinline__ void tc_commit(uint32_t bar, int lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead)
      : "memory");
}
// 32 consecutive columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
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
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
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
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
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
// The products' warp stays together and one lane (`lead`) issues: operands that
// are the same for the whole warp are in uniform registers then, where the
// instruction wants them.  (Issued from a branch of one lane, every operand is
// moved there first, and four products take 660 cycles to issue.)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t word, bool add, int lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(word),
      "r"((int)add), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t word, bool add, int lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(word),
      "r"((int)add), "r"(lead)
      : "memory");
}
__device__ __forceinline__ int elect_one() {
  int r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// A load that stays where it is issued, ahead of its use (a plain read-only load
// is moved down to it by the compiler).
__device__ __forceinline__ int64_t ld_ahead8(const void* p) {
  int64_t r;
  asm volatile("ld.global.nc.s64 %0, [%1];" : "=l"(r) : "l"(p));
  return r;
}

// Two float32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, __half2 f) {
  const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&a), f);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Byte offset of 16-byte chunk `c` of a row's 64-column panel in a swizzled tile of `rows` rows.
__device__ __forceinline__ uint32_t swz(int rows, int row, int panel, int c) {
  return (uint32_t)(panel * (rows * 128) + row * 128 + ((c ^ (row & 7)) << 4));
}
// Waits of all roles: bounded, and given up when another role has given up.
__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* stop, int* err) {
  for (int n = 0; n < kWaitSpinLimit; ++n) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((n & 63) == 63 && *stop) return false;
  }
  *stop = 1;
  atomicOr(err, MVB_DEV_TIMEOUT);
  return false;
}
struct Waiter {
  uint32_t bars;
  volatile int* stop;
  int* err;
  __device__ __forceinline__ uint32_t bar(int i) const { return bars + 8 * i; }
  // All lanes of a warp, which stay together whatever each of them saw.
  __device__ __forceinline__ bool warp(int i, int parity) const {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar(i), (uint32_t)parity))) return true;
    return __all_sync(0xffffffffu, wait_on(bar(i), (uint32_t)parity, stop, err)) != 0;
  }
};

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
  float* const sums = a.part + (int64_t)a.splits * a.total_q * a.num_heads * D;
  auto part_row = [&](int r) {  // of the chunk's row r in this CTA's partial results
    return ((int64_t)blockIdx.z * a.total_q + q0 + r / a.G) * a.num_heads + h0 + r % a.G;
  };
  auto nothing = [&]() {  // this CTA adds nothing to its rows
    for (int r = tid; r < nrows; r += kThreads) sums[part_row(row0 + r)] = -INFINITY;
  };
  const int64_t srow = __ldg(a.seq_rows + lo), cached = __ldg(a.cached + lo);
  T* const out = static_cast<T*>(a.out);
  if (cached < 0 || cached > (int64_t)a.max_blocks << a.block_shift || srow < 0 || srow >= a.bt_rows ||
      (cached + ql + (1 << a.block_shift) - 1) >> a.block_shift > a.max_blocks) {
    // a table too short for the chunk (or a bad row): zeros, and the flag
    if (tid == 0) atomicOr(a.err, MVB_DEV_TABLE_SHORT);
    if (a.splits > 1) nothing();
    for (int e = tid; e < nrows * D && a.splits == 1; e += kThreads) {
      const int r = row0 + e / D;
      out[(int64_t)(q0 + r / a.G) * a.o_s0 + (int64_t)(h0 + r % a.G) * a.o_s1 + e % D] = from_f32<T>(0.f);
    }
    return;
  }
  int kv_end = (int)cached + (row0 + nrows - 1) / a.G + 1;  // positions the CTA's last row attends
  int steps = (kv_end + kKeys - 1) / kKeys, first = 0;      // this CTA's steps, and its first position
  if (a.splits > 1) {
    const int share = max(kMinSteps, (steps + a.splits - 1) / a.splits), from = (int)blockIdx.z * share;
    if (from >= steps) {
      nothing();
      return;
    }
    steps = min(share, steps - from);
    first = from * kKeys;
    kv_end = min(kv_end - first, steps * kKeys);  // relative to first, as all positions below
  }
  const int tiles = (nrows + kTileRows - 1) / kTileRows;

  Waiter wait;
  wait.bars = smem_u32(smem + G_::BARS);
  wait.stop = &s_stop;
  wait.err = a.err;
  StepInfo* infos = reinterpret_cast<StepInfo*>(smem + G_::INFO);
  uint16_t* masks = reinterpret_cast<uint16_t*>(smem + G_::MASK);  // [kMasks][kKeys][D / 16]
  if (warp == kMmaWarp) tmem_alloc(smem_u32(&s_tmem));
  if (tid == 0) {
    s_stop = 0;
    mbar_init(wait.bar(kQ), 4 * tiles);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(wait.bar(kKFull + i), 4);
      mbar_init(wait.bar(kVFull + i), 4);
      mbar_init(wait.bar(kKEmpty + i), tiles);
      mbar_init(wait.bar(kVEmpty + i), tiles);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(wait.bar(kSFull + i), 1);
      mbar_init(wait.bar(kPReady + i), 4);
      mbar_init(wait.bar(kPvDone + i), 1);
      mbar_init(wait.bar(kGivenUp + i), 1);
    }
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  if (warp < kLoadWarp) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G_::SOFTMAX));
    // ================================ softmax =================================
    const int tile = warp >> 2, r0 = row0 + tile * kTileRows + (warp & 3) * 32 + lane;
    if (tile < tiles) {
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t o_at = tmem + lanes + G_::O_COL + tile * D;
      const bool live = r0 < rows;
      const int tok = live ? r0 / a.G : 0, head = live ? r0 - tok * a.G : 0;
      const int lim = live ? (int)cached + tok + 1 - first : kv_end;  // rows past the chunk are zeros that attend all
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
          *reinterpret_cast<uint4*>(qd + swz(kTileRows, qr, i / 8, i % 8)) = w;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(wait.bar(kQ));
      }
      float m = -INFINITY, l = 0.f;
      uint32_t nanbits[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) nanbits[i] = 0u;
      auto take_nan = [&](int j) {  // columns of step j's values that are NaN for this row
        const StepInfo& f = infos[j % kInfos];
        if (!(f.nan[0] | f.nan[1] | f.nan[2] | f.nan[3])) return;
        const int n = min(kKeys, lim - j * kKeys);
        for (int k = 0; k < n; ++k)
          if (f.nan[k / (512 / D) & 3])  // the warp that loaded the key
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
              nanbits[i] |= reinterpret_cast<const uint32_t*>(masks + ((j % kMasks) * kKeys + k) * (D / 16))[i];
      };
      enum { kLeave, kDone, kAnew };  // a wait ran out; the step is done; it wants its maximum taken anew
      // One step of the softmax.  EDGE: it takes its maximum anew, or holds keys that some row does not attend
      // (`masked`); one form for both: with the second pass in each form, 8192 tokens took 293 us for 275.
      auto step = [&](int j, auto edge, bool anew, bool masked, float rf) {
        constexpr bool EDGE = decltype(edge)::value;
        const StepInfo& f = infos[j % kInfos];
        const int rem = lim - j * kKeys;
        const uint32_t s_at = tmem + lanes + (tile * NB + j % NB) * kKeys;  // P goes over it
        // columns read at a time, two reads in flight; P waits in registers until the step holds
        constexpr int CW = 16, NC = kKeys / CW;
        uint32_t s[2][CW];
        auto read = [&](int h) {
          tmem_ld16(s_at + CW * h, s[h & 1]);
        };
        auto mask = [&](int h) {  // -inf where the row does not attend the key
          if (EDGE && masked) {
            const int bad = f.bad >> (CW / 16 * h), n = rem - CW * h;
#pragma unroll
            for (int i = 0; i < CW; ++i)
              if (i >= n || (bad >> (i / 16) & 1)) s[h & 1][i] = 0xff800000u;
          }
        };
        auto factor = [&](float ks) { return fmaxf(qs * ks, 1.2e-38f); };  // (not 0: -inf stays -inf)
        float fac = rf;
        bool move = rf != 1.f;
        // P against the maximum at hand; whether 16 of them add up to more than 2^14
        uint32_t p[kKeys / 2];
        float sum = 0.f;
        auto weights = [&]() {
          read(NC - 1);
          float4 info[2][CW / 16];  // of the columns at hand and of the next ones
#pragma unroll
          for (int g = 0; g < CW / 16; ++g) info[(NC - 1) & 1][g] = f.g[CW / 16 * (NC - 1) + g];
          float most = 0.f;
#pragma unroll
          for (int h = NC - 1; h >= 0; --h) {
            const uint32_t(&x)[CW] = s[h & 1];
            tc_wait_ld();
            if (h > 0) {
              read(h - 1);
#pragma unroll
              for (int g = 0; g < CW / 16; ++g) info[(h - 1) & 1][g] = f.g[CW / 16 * (h - 1) + g];
            }
            mask(h);
#pragma unroll
            for (int gg = 0; gg < CW / 16; ++gg) {
              const float4 in = info[h & 1][gg];
              const float c = factor(in.x), b = in.y - m;
              const float2 cc = make_float2(c, c), mm = make_float2(b, b);
              float2 t[2];
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                float2 e = fma2(make_float2(__uint_as_float(x[16 * gg + i]), __uint_as_float(x[16 * gg + i + 1])), cc, mm);
                e.x = fast_exp2(e.x);
                e.y = fast_exp2(e.y);
                t[i / 2 & 1] = i < 4 ? e : add2(t[i / 2 & 1], e);
                p[CW / 2 * h + 8 * gg + i / 2] = pack_h2(e.x, e.y);
              }
              t[0] = add2(t[0], t[1]);
              const float u = t[0].x + t[0].y;
              most = fmaxf(most, u);
              sum = fmaf(u, in.z, sum);
            }
          }
          return most > 16384.f;
        };
        const bool holds = !anew && !__any_sync(0xffffffffu, weights());
        if (!EDGE && !holds) return kAnew;
        if (!EDGE || holds) {
          tmem_st16(s_at, p);
          tmem_st16(s_at + 16, p + 16);
        } else {
          float mx = m;
#pragma unroll
          for (int h = 0; h < NC; ++h) {
            if (h == 0) read(0);
            tc_wait_ld();
            if (h + 1 < NC) read(h + 1);
            mask(h);
#pragma unroll
            for (int g = 0; g < CW / 16; ++g) {
              float top = -INFINITY;
#pragma unroll
              for (int i = 0; i < 16; i += 2)
                top = fmaxf(fmaxf(top, __uint_as_float(s[h & 1][16 * g + i])), __uint_as_float(s[h & 1][16 * g + i + 1]));
              mx = fmaxf(mx, __fmul_rn(top, factor(f.g[CW / 16 * h + g].x)));
            }
          }
          const float al = mx == m ? 1.f : fast_exp2(m - mx);  // (0 for a row's first keys, where l and O are 0)
          m = mx;
          l *= al;
          fac *= al;
          move = true;
          // The exponents above are fused multiply-adds: their products are not rounded, so they can lie half an ulp of
          // m above the maximum of the rounded ones (2^4 from |m| = 2^28 on).  Against this maximum they are therefore
          // differences of the rounded ones: 0 at the largest, nowhere above the group's part of the value scale (2^7),
          // whatever the logits' size.  (A row that has attended nothing yet: m and all of s are -inf, and P is 0.)
          const float base = m == -INFINITY ? 0.f : -m;
          sum = 0.f;
          static_assert(CW == 16, "a group's P covers scores that have been read");
#pragma unroll
          for (int h = 0; h < NC; ++h) {
            if (h == 0) read(0);
            const float4 in = f.g[h];
            const float c = factor(in.x);
            const float2 mm = make_float2(base, base), vv = make_float2(in.y, in.y);
            tc_wait_ld();
            if (h + 1 < NC) read(h + 1);
            mask(h);
            float2 t = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              // (packed products are joined with the sum behind them, for all their rounding modes)
              float2 e = make_float2(__fmul_rn(__uint_as_float(s[h & 1][i]), c), __fmul_rn(__uint_as_float(s[h & 1][i + 1]), c));
              e = add2(add2(e, mm), vv);
              e.x = fast_exp2(e.x);
              e.y = fast_exp2(e.y);
              t = add2(t, e);
              p[i / 2] = pack_h2(e.x, e.y);
            }
            sum = fmaf(t.x + t.y, in.z, sum);
            tmem_st8(s_at + 8 * h, p);
          }
        }
        l += sum;
        if (move && j > 0) {
          // the last step's products add to O
          if (!wait.warp(kPvDone + tile * NB + (j - 1) % NB, ((j - 1) / NB) & 1)) return kLeave;
          tc_fence_after();
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
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(wait.bar(kPReady + tile * NB + j % NB));
        return kDone;
      };
      const int least = __reduce_min_sync(0xffffffffu, lim);
      bool ok = true, fresh = true;
      for (int j = 0; ok && j < steps; ++j) {
        // before the wait: what is known of the step (the scores of the one before it came after the loaders had
        // written it) and the NaN of values whose products are done (those scores came after them)
        const bool edge = least - j * kKeys < kKeys;
        if (fresh) fresh = __any_sync(0xffffffffu, m == -INFINITY);  // a row's first keys
        if (j >= kNanLag) take_nan(j - kNanLag);
        if (j == 0 && !wait.warp(kSFull + tile * NB, 0)) break;
        const float rf = infos[j % kInfos].rf;
        const int bad = infos[j % kInfos].bad;
        ok = wait.warp(kSFull + tile * NB + j % NB, (j / NB) & 1);
        if (!ok) break;
        tc_fence_after();
        const bool masked = edge || bad;
        int did = masked || fresh ? kAnew : step(j, std::false_type(), false, false, rf);
        if (did == kAnew) did = step(j, std::true_type(), fresh || !masked, masked, rf);
        ok = did == kDone;
      }
      if (ok && wait.warp(kPvDone + tile * NB + (steps - 1) % NB, ((steps - 1) / NB) & 1)) {
        tc_fence_after();
        for (int j = max(0, steps - kNanLag); j < steps; ++j) take_nan(j);
        const float inv = l == 0.f ? 0.f : infos[(steps - 1) % kInfos].r / l;
        int r = r0;
        asm("" : "+r"(r));  // (the row's place, worked out again and not kept in registers through the steps)
        const bool live = r < rows;
        const int tok = live ? r / a.G : 0, head = live ? r - tok * a.G : 0;
        float4* const pp = reinterpret_cast<float4*>(a.part + (a.splits > 1 ? part_row(live ? r : 0) * D : 0));
        if (a.splits > 1 && live) sums[part_row(r)] = l == 0.f ? -INFINITY : m + log2f(l);
        T* op = out + (int64_t)(q0 + tok) * a.o_s0 + (int64_t)(h0 + head) * a.o_s1;
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
          uint32_t o[32];
          tmem_ld32(o_at + 32 * h, o);
          tc_wait_ld();
          if (!live) continue;
          if (a.splits > 1) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              o[i] = (nanbits[h] >> i) & 1 ? 0x7fffffffu : __float_as_uint(__uint_as_float(o[i]) * inv);
#pragma unroll
            for (int i = 0; i < 8; ++i) pp[8 * h + i] = reinterpret_cast<const float4*>(o)[i];
            continue;
          }
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
  } else if (warp < kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G_::LOADER));
    // ================================ loaders =================================
    constexpr int CH = D / 16, N = kKeys * CH / 128;  // 16-code chunks per row, chunks per thread and tile
    constexpr uint32_t NONE = 0xffffffffu, IN_STEP = (1u << kGroups) - 1;
    const bool is_v = warp >= kLoadWarp + 4;
    const int lw = warp & 3;
    const int64_t* bt = a.bt + srow * a.bt_s0;
    const int BSm = (1 << a.block_shift) - 1, gshift = a.block_shift - 4;
    // kBatch steps at a time, one 16-key group per lane: its number among the cache's groups (NONE behind the last
    // key or for a bad block id), and its block's scales.
    auto find = [&](int j0, bool& bad) {
      int p = j0 * kKeys + 16 * lane;
      bad = false;
      if (p >= kv_end) return NONE;
      p += first;
      const int64_t b = ld_ahead8(bt + (p >> a.block_shift));
      bad = b < 0 || b >= a.num_blocks;
      return bad ? NONE : ((uint32_t)(b * a.num_kv_heads + kvh) << gshift) + ((uint32_t)(p & BSm) >> 4);
    };
    auto scales = [&](uint32_t group) {
      const int64_t v = group != NONE ? ld_ahead8(a.scale + (group >> gshift)) : 0;
      return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
    };
    // This thread's chunk i of a step: key key0 + i * (128 / CH), codes [16 ch, 16 ch + 16).  Eight lanes hold the
    // chunks of one panel of two keys, whose swizzled places are in different banks.
    const int ch = CH == 4 ? lane & 3 : (lane & 3) | (lane >> 1 & 4);
    const int key0 = CH == 4 ? lw * 8 + (lane >> 2) : lw * 4 + ((lane >> 2 & 1) | (lane >> 3 & 2));
    uint8_t* const raw = smem + G_::RAW + (is_v ? G_::RAWBYTES : 0) + (lw * 32 + lane) * 16;  // its codes: + 2048 i
    const uint32_t to0 = swz(kKeys, key0, ch / 4, 2 * (ch % 4)), to1 = to0 ^ 16;  // its places in a tile: + i * STEP
    constexpr uint32_t STEP = (128 / CH) * 128;
    const uint8_t* const base = (is_v ? a.vc : a.kc) + (key0 & 15) * D + ch * 16;
    const uint32_t dst = smem_u32(raw);
    auto fetch = [&](int j, uint32_t groups) {
      const bool tail = (j + 1) * kKeys > kv_end;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int key = key0 + i * (128 / CH);
        const uint32_t grp = __shfl_sync(0xffffffffu, groups, (j % kBatch) * kGroups + (key >> 4));
        const bool ok = grp != NONE && !(tail && j * kKeys + key >= kv_end);
        cp_async_16(dst + 2048 * i, base + (ok ? (uint64_t)grp * (16 * D) : 0), ok ? 16 : 0);
      }
      cp_async_commit();
    };
    bool bad, bad_n;
    uint32_t grp = find(0, bad), grp_n = find(kBatch, bad_n);
    fetch(0, grp);
    const float2 sc = scales(grp);
    float2 sc_n = make_float2(0.f, 0.f);
    int RE = 0;          // exponent field of R (0: no value scale has given it yet)
    uint32_t rests = 0;  // lanes whose group's value scale goes into the codes in part
    float rest = 1.f;
    // The side information of kBatch steps from j on; each lane's part of its group's scale that goes into the codes
    // of V, and the lanes where that is not 1.
    auto side_info = [&](int j, float2 sc, uint32_t grp, bool bad, float& rest, uint32_t& rests) {
      const int vexp = (int)(__float_as_uint(sc.y) >> 23) & 0xff;  // 0: a scale of 0 or below 2^-126
      int top = vexp, mine = 127;  // largest exponent field of the step; R's of this lane's step
      float rf = 1.f;
#pragma unroll
      for (int o = 1; o < kGroups; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll 1
      for (int k = 0; k < kBatch; ++k) {
        const int t = __shfl_sync(0xffffffffu, top, k * kGroups);
        const int was = RE;
        if (RE == 0 || t > RE + 7) RE = t;
        if (lane / kGroups == k && RE > 0) {  // (before that O is 0, in any unit)
          mine = RE;
          if (was > 0 && RE != was) rf = RE - was < 127 ? __uint_as_float((uint32_t)(127 + was - RE) << 23) : 0.f;
        }
      }
      const int e = vexp > 0 ? vexp - mine : 0, ep = max(e, kMinValueExp);
      rest = grp != NONE && vexp == 0 ? 0.f
             : e == ep                ? 1.f
             : e - ep > -127          ? __uint_as_float((uint32_t)(127 + e - ep) << 23)
                                      : 0.f;
      rests = __ballot_sync(0xffffffffu, rest != 1.f);
      const uint32_t bads = __ballot_sync(0xffffffffu, bad);
      if (!is_v && lw == 0) {
        const float vf = vexp > 0 ? __uint_as_float((__float_as_uint(sc.y) & 0x7fffffu) | 0x3f800000u) : 1.f;
        StepInfo& f = infos[(j + lane / kGroups) % kInfos];
        const int g = lane % kGroups;
        float ve = (float)ep, vu = __uint_as_float((uint32_t)(127 - ep) << 23);
        if (vf != 1.f) {
          ve += log2f(vf);
          vu /= vf;
        }
        f.g[g] = make_float4(sc.x, ve, vu, 0.f);
        if (g == 0) {
          f.r = __uint_as_float((uint32_t)mine << 23);
          f.rf = rf;
          f.bad = (int)(bads >> (lane & ~(kGroups - 1)) & IN_STEP);
        }
        if (lane == 0 && bads) atomicOr(a.err, MVB_DEV_BLOCK_ID);
      }
      __syncwarp();
    };
    uint32_t rests_n = 0;
    float rest_n = 1.f;
    side_info(0, sc, grp, bad, rest, rests);
    for (int j = 0; j < steps; ++j) {
      const int st = j % kStages, q = (j % kBatch) * kGroups;
      const int again = (j / kStages - 1) & 1;  // parity of the stage's last use
      if (q == (kBatch - 1) * kGroups) side_info(j + 1, sc_n, grp_n, bad_n, rest_n, rests_n);
      const uint32_t groups_next = (j + 1) % kBatch == 0 ? grp_n : grp;
      if (!is_v) {
        if (j >= kStages && !wait.warp(kKEmpty + st, again)) break;
        cp_async_wait<0>();
        uint8_t* tile = smem + G_::K + st * G_::KBYTES;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint4 x = *reinterpret_cast<const uint4*>(raw + 2048 * i);
          uint4 lo4, hi4;
          e4m3x4_to_f16(x.x, lo4.x, lo4.y);
          e4m3x4_to_f16(x.y, lo4.z, lo4.w);
          e4m3x4_to_f16(x.z, hi4.x, hi4.y);
          e4m3x4_to_f16(x.w, hi4.z, hi4.w);
          *reinterpret_cast<uint4*>(tile + to0 + i * STEP) = lo4;
          *reinterpret_cast<uint4*>(tile + to1 + i * STEP) = hi4;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(wait.bar(kKFull + st));
      } else {
        if (j >= kStages && !wait.warp(kVEmpty + st, again)) break;
        cp_async_wait<0>();
        uint8_t* tile = smem + G_::V + st * G_::KBYTES;
        uint32_t seen = 0;
        auto store = [&](uint4 x, int i) {
          uint4 lo4, hi4;
          e4m3x4_to_f16(x.x, lo4.x, lo4.y);
          e4m3x4_to_f16(x.y, lo4.z, lo4.w);
          e4m3x4_to_f16(x.z, hi4.x, hi4.y);
          e4m3x4_to_f16(x.w, hi4.z, hi4.w);
          if (rests >> q & IN_STEP) {
            const __half2 r2 =
                __float2half2_rn(__shfl_sync(0xffffffffu, rest, q + ((key0 + i * (128 / CH)) >> 4)));
            lo4 = make_uint4(mul_h2(lo4.x, r2), mul_h2(lo4.y, r2), mul_h2(lo4.z, r2), mul_h2(lo4.w, r2));
            hi4 = make_uint4(mul_h2(hi4.x, r2), mul_h2(hi4.y, r2), mul_h2(hi4.z, r2), mul_h2(hi4.w, r2));
          }
          *reinterpret_cast<uint4*>(tile + to0 + i * STEP) = lo4;
          *reinterpret_cast<uint4*>(tile + to1 + i * STEP) = hi4;
        };
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint4 x = *reinterpret_cast<const uint4*>(raw + 2048 * i);
          // a byte 0x7f or 0xff is NaN: its low seven bits and one more reach the eighth
          seen |= ((x.x & 0x7f7f7f7fu) + 0x01010101u) | ((x.y & 0x7f7f7f7fu) + 0x01010101u) |
                  ((x.z & 0x7f7f7f7fu) + 0x01010101u) | ((x.w & 0x7f7f7f7fu) + 0x01010101u);
          store(x, i);
        }
        const bool any_nan = __any_sync(0xffffffffu, (seen & 0x80808080u) != 0);
        if (any_nan) {  // once more with zeros in their place, and the masks
#pragma unroll 1
          for (int i = 0; i < N; ++i) {
            uint4 x = *reinterpret_cast<const uint4*>(raw + 2048 * i);
            uint32_t* w = reinterpret_cast<uint32_t*>(&x);
            uint32_t nan16 = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t n = ((w[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
              w[k] &= ~((n >> 7) * 0xffu);
              nan16 |= ((n >> 7 & 1) | (n >> 14 & 2) | (n >> 21 & 4) | (n >> 28 & 8)) << (4 * k);
            }
            masks[((j % kMasks) * kKeys + key0 + i * (128 / CH)) * CH + ch] = (uint16_t)nan16;
            store(x, i);
          }
        }
        if (lane == 0) infos[j % kInfos].nan[lw] = any_nan;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(wait.bar(kVFull + st));
      }
      fetch(j + 1, groups_next);  // nothing behind the last key
      if (j % kBatch == kBatch / 2 - 1) sc_n = scales(grp_n);
      if (j % kBatch == kBatch - 1) {
        grp = grp_n;
        rest = rest_n;
        rests = rests_n;
        grp_n = find(j + 1 + kBatch, bad_n);
      }
    }
    cp_async_wait<0>();  // nothing lands after the CTA has left
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G_::MMA));
    // ==================== tensor-core products of row tile i ====================
    const int i = warp - kMmaWarp;
    if (i < tiles) {
      const uint32_t base = smem_u32(smem);
      const int lead = elect_one();
      constexpr uint32_t SW = mma_word(kKeys, false), PW = mma_word(D, true);
      const uint32_t s_col = tmem + i * NB * kKeys, o_col = tmem + G_::O_COL + i * D;
      auto scores = [&](int j) {  // S = Q K^T of step j: 16 columns (32 bytes of a panel's row) at a time
        const uint64_t qd = smem_desc(base + G_::Q + i * G_::QBYTES, 16, 1024);
        const uint64_t kd = smem_desc(base + G_::K + (j % kStages) * G_::KBYTES, 16, 1024);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          mma_ss(s_col + (j % NB) * kKeys, qd + (((k / 4) * (kTileRows * 128) + (k % 4) * 32) >> 4),
                 kd + (((k / 4) * (kKeys * 128) + (k % 4) * 32) >> 4), SW, k > 0, lead);
        tc_commit(wait.bar(kSFull + i * NB + j % NB), lead);
        tc_commit(wait.bar(kKEmpty + j % kStages), lead);
      };
      auto values = [&](int j) {  // O += P V of step j: 16 keys (2 KB of a panel) at a time
        const uint64_t vd = smem_desc(base + G_::V + (j % kStages) * G_::KBYTES, kKeys * 128, 1024);
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          mma_ts(o_col, s_col + (j % NB) * kKeys + 8 * k, vd + (k * 2048 >> 4), PW, j > 0 || k > 0, lead);
        tc_commit(wait.bar(kPvDone + i * NB + j % NB), lead);
        tc_commit(wait.bar(kVEmpty + j % kStages), lead);
      };
      auto ready = [&](int b, int parity) {
        if (!wait.warp(b, parity)) return false;
        tc_fence_after();
        return true;
      };
      auto ready_k = [&](int j) { return ready(kKFull + j % kStages, (j / kStages) & 1); };
      bool ok = ready(kQ, 0);
      for (int j = 0; ok && j < min(NB, steps); ++j) {
        ok = ready_k(j);
        if (ok) scores(j);
      }
      for (int j = 0; ok && j < steps; ++j) {
        ok = ready(kVFull + j % kStages, (j / kStages) & 1) && ready(kPReady + i * NB + j % NB, (j / NB) & 1);
        if (!ok) break;
        values(j);
        if (j + NB < steps) {  // S overwrites P: the products that read it come first
          ok = ready_k(j + NB) && ready(kPvDone + i * NB + j % NB, (j / NB) & 1);
          if (ok) scores(j + NB);
        }
      }
      if (!ok) {  // given up: wait for whatever was issued before the tensor memory goes
        tc_commit(wait.bar(kGivenUp + i), lead);
        mbar_wait_bounded(wait.bar(kGivenUp + i), 0);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_free(tmem);
}

// Joins the CTAs' results of a row: out = sum of w_z O_z / sum of w_z, w_z = 2^(sums_z - their maximum).  D / 4
// threads per row; a few MB that are still in L2.
template <typename T, int D>
__global__ void __launch_bounds__(128) fp8_prefill_merge_kernel(const Fp8PrefillArgs a) {
  __shared__ int s_n[4];
  const int tid = threadIdx.x;
  grid_dependency_wait();
  grid_launch_dependents();
  int have = 0;  // tokens of all chunks: rows behind them stay
  for (int i = tid; i < a.n; i += 128)
    have = min(have + (int)min((int64_t)a.total_q + 1, max((int64_t)0, __ldg(a.qlen + i))), a.total_q + 1);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) have = min(have + __shfl_xor_sync(0xffffffffu, have, o), a.total_q + 1);
  if (tid % 32 == 0) s_n[tid / 32] = have;
  __syncthreads();
  have = min(min(s_n[0] + s_n[1], a.total_q + 1) + min(s_n[2] + s_n[3], a.total_q + 1), a.total_q + 1);
  if (have > a.total_q) return;  // refused by the kernel before
  constexpr int TPR = D / 4;
  const int64_t rows = (int64_t)a.total_q * a.num_heads, row = (int64_t)blockIdx.x * (128 / TPR) + tid / TPR;
  if (row >= (int64_t)have * a.num_heads) return;
  const int c = tid % TPR;
  const float* sums = a.part + a.splits * rows * D;
  float top = -INFINITY;
  for (int z = 0; z < a.splits; ++z) top = fmaxf(top, sums[z * rows + row]);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int z = 0; z < a.splits; ++z) {
    const float s = sums[z * rows + row];
    if (s == -INFINITY) continue;  // nothing was written there
    const float w = fast_exp2(s - top);
    const float4 o = reinterpret_cast<const float4*>(a.part + (z * rows + row) * D)[c];
    acc = make_float4(fmaf(w, o.x, acc.x), fmaf(w, o.y, acc.y), fmaf(w, o.z, acc.z), fmaf(w, o.w, acc.w));
    l += w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint2 w;
  T* e = reinterpret_cast<T*>(&w);
  e[0] = from_f32<T>(acc.x * inv);
  e[1] = from_f32<T>(acc.y * inv);
  e[2] = from_f32<T>(acc.z * inv);
  e[3] = from_f32<T>(acc.w * inv);
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (row / a.num_heads) * a.o_s0 + (row % a.num_heads) * a.o_s1 +
                            4 * c) = w;
}

int64_t row_tiles(int total_q, int G, int num_chunks) {  // at most
  return ((int64_t)total_q * G + kCtaRows - 1) / kCtaRows + num_chunks;
}

// How many CTAs share a row tile's keys: as many as there are SMs for, each with kMinSteps steps or more.  With one
// CTA and shared (14/2 heads of 64): 20 tokens after 300: 13.7 and 14.4 us, 20 after 600: 20.1 and 14.6, 37 after
// 1003: 30.1 and 17.5, 512 after 32768: 646 and 175; with four steps or more, 13.8, 17.3, 19.3 and 175.
int num_splits(int64_t ctas, int64_t max_keys) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t steps = (max_keys + kKeys - 1) / kKeys;
  const int64_t most = std::min(sms / ctas, std::min<int64_t>(steps / kMinSteps, kMaxSplits));
  return most > 1 ? (int)most : 1;
}

template <typename T, int D>
int launch_prefill_fp8(const Fp8PrefillArgs& a, cudaStream_t stream) {
  static_assert(2 * (kFp8PrefillMaxChunks + 1) * 4 <= 2 * kStages * Geo<D>::KBYTES, "the prefixes fit the stages");
  static_assert(Geo<D>::BYTES <= 227 * 1024 - 512, "shared memory of one CTA");
  const int64_t tiles = row_tiles(a.total_q, a.G, a.n);
  auto kern = fp8_prefill_kernel<T, D>;
  if (ensure_kernel_attrs(kern, Geo<D>::BYTES) != cudaSuccess) return MVB_ERR_CUDA;
  if (launch_pdl(kern, dim3((unsigned)tiles, a.num_kv_heads, a.splits), dim3(kThreads), Geo<D>::BYTES, stream, a) !=
      cudaSuccess)
    return MVB_ERR_CUDA;
  if (a.splits == 1) return MVB_OK;
  auto merge = fp8_prefill_merge_kernel<T, D>;
  if (ensure_kernel_attrs(merge, 0) != cudaSuccess) return MVB_ERR_CUDA;
  const int64_t rows = (int64_t)a.total_q * a.num_heads, per = 128 / (D / 4);
  return launch_pdl(merge, dim3((unsigned)((rows + per - 1) / per)), dim3(128), 0, stream, a) == cudaSuccess
             ? MVB_OK
             : MVB_ERR_CUDA;
}

}  // namespace
}  // namespace mvb

using namespace mvb;

namespace {
int plan_prefill(int num_chunks, int total_q, int num_heads, int num_kv_heads, int head_dim, int block_size,
                 int max_blocks, int* splits, int64_t* bytes) {
  if (head_dim != 64 && head_dim != 128) return MVB_ERR_HEAD_DIM;
  if (block_size < kFp8MinBlock || block_size > kFp8MaxBlock || (block_size & (block_size - 1)) != 0)
    return MVB_ERR_BLOCK_SIZE;
  if (num_chunks < 0 || num_chunks > kFp8PrefillMaxChunks || total_q < 0 || num_heads <= 0 || num_kv_heads <= 0 ||
      num_kv_heads > 65535 || max_blocks < 0)
    return MVB_ERR_INVALID_ARG;
  if (num_heads % num_kv_heads != 0) return MVB_ERR_HEADS;
  const int G = num_heads / num_kv_heads;
  // rows of a KV head and positions of a sequence are 32-bit
  if ((int64_t)total_q * G >= ((int64_t)1 << 30) || (int64_t)max_blocks * block_size >= ((int64_t)1 << 30))
    return MVB_ERR_INVALID_ARG;
  *splits = 1;
  *bytes = 0;
  if (num_chunks == 0 || total_q == 0) return MVB_OK;
  *splits = num_splits(row_tiles(total_q, G, num_chunks) * num_kv_heads, (int64_t)max_blocks * block_size);
  if (*splits > 1) *bytes = (int64_t)*splits * total_q * num_heads * (head_dim + 1) * 4;
  return MVB_OK;
}
}  // namespace

extern "C" int mvb_paged_prefill_fp8_workspace(int32_t num_chunks, int32_t total_q, int32_t num_heads,
                                               int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                               int32_t max_blocks_per_seq, int64_t* bytes_out) {
  int splits = 1;
  int64_t bytes = 0;
  const int st = plan_prefill(num_chunks, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                              &splits, &bytes);
  if (st == MVB_OK && bytes_out) *bytes_out = bytes;
  return st;
}

extern "C" int mvb_paged_prefill_fp8(const void* query, int64_t q_stride_tok, int64_t q_stride_head,
                                     const void* key_cache, const void* value_cache, const float* kv_scale,
                                     const int64_t* block_table, int64_t block_table_rows,
                                     int64_t block_table_stride, int32_t max_blocks_per_seq, const int64_t* seq_rows,
                                     const int64_t* cached_len, const int64_t* query_len, int32_t num_chunks,
                                     int32_t total_q, void* out, int64_t out_stride_tok, int64_t out_stride_head,
                                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                     int32_t num_blocks, float scale, int32_t dtype, void* workspace,
                                     int64_t workspace_bytes, int32_t* error_flags, void* stream) {
  mvb::NvtxRange nvtx_range("mvb_paged_prefill_fp8");
  if (dtype != MVB_DTYPE_F16 && dtype != MVB_DTYPE_BF16) return MVB_ERR_DTYPE;
  int splits = 1;
  int64_t bytes = 0;
  const int st = plan_prefill(num_chunks, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                              &splits, &bytes);
  if (st != MVB_OK) return st;
  if (num_blocks <= 0 || block_table_rows < 0) return MVB_ERR_INVALID_ARG;
  // (block, KV head) and 16-token group numbers are 32-bit
  if ((int64_t)num_blocks * num_kv_heads >= ((int64_t)1 << 31) ||
      (int64_t)num_blocks * num_kv_heads * (block_size / 16) >= 0xffffffffll)
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
  if (bytes > 0 && (workspace == nullptr || workspace_bytes < bytes || !al(workspace, 256))) return MVB_ERR_WORKSPACE;
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
  a.G = num_heads / num_kv_heads;
  a.block_shift = 31 - __builtin_clz(block_size);
  a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.splits = splits;
  a.part = static_cast<float*>(workspace);
  a.err = error_flags;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MVB_DTYPE_BF16)
    return head_dim == 64 ? launch_prefill_fp8<__nv_bfloat16, 64>(a, s) : launch_prefill_fp8<__nv_bfloat16, 128>(a, s);
  return head_dim == 64 ? launch_prefill_fp8<__half, 64>(a, s) : launch_prefill_fp8<__half, 128>(a, s);
}
