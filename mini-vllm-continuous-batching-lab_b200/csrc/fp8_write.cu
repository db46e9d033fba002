// mvb_rope_kv_cache_write_fp8: rotary embedding of a step's queries and keys
// and the write of the rotated keys and the values into an 8-bit paged cache
// whose scales belong to (block, KV head).  Without the rotation it is the
// plain write.
//
// What a call does to a block b it writes to, for each KV head and for keys and
// values apart (x: the call's rows in float32, keys after the rotation):
//   base  = 0 if the call writes slot 0 of b (the block starts anew), else b's scale
//   s     = max(base, the smallest power of two that maps max |x| into 448)
//   codes of the block's other rows = round(code * base / s)   where s > base > 0
//   codes of the rows x             = round(x / s)
// round is to the nearest e4m3 value, ties to even.  With powers of two the
// quotients are exact, so rows that are rounded anew keep their values except
// where these fall below the smallest normal code (2^-6 s), and what a block
// holds does not depend on how its tokens were split into calls but for those.
// The maximum runs over the finite elements; an infinity is stored as +-448 s.
//
// Queries and returned keys are a product and a fused multiply-add in float32.
// With float32 tables the product is rounded, so beside a tie one code in 2^20
// would differ from the exact rotation's: the keys are coded from sums with their
// rounding errors added back (rope_exact; 63.7 against 60.8 us for the chunks
// below).  Their maximum is taken without; only one within 4 ulps of 448 * 2^k
// decides about a scale, and there it is taken again.
//
// Work split.  A block's scale needs the maximum over all the call's rows of the
// block, so its rows belong together, with the CTA of the block's leader: the
// token that writes the block's lowest slot of the call.  A warp takes one (KV
// head, keys or values) and all of the block's rows at once, D / 16 lanes a row;
// where the call writes a single row (a decode step), each D / 16 lanes take a
// (KV head, keys or values) of their own.  Leaders are found in one of two ways:
//   * up to kFp8ScanTokens tokens, each token's CTA reads every slot of the call
//     and keeps the rows of its block in shared memory: one launch;
//   * more tokens: a first kernel stores writer[slot] = token, and a CTA reads
//     the entries of its eight tokens' blocks.  An entry is believed only if
//     slot_mapping[entry] is that slot, so the array needs no initialisation and
//     keeps nothing from one call to the next.
// The query rows are rotated by CTAs of their own, behind the others in the same
// launch: a thread holds 8 + 8 columns of two heads of one token (four, where there
// are many tokens), so the cos and sin rows are read once for them.
// Bound: memory for long chunks; for a decode step the latency of slots ->
// rows -> maximum -> codes.  Measured: 9721 tokens of 32/8 heads of 128, 229 MB:
// 64 us, 3.6 TB/s (latency at 16 warps an SM: 38 % of the issue slots are used; each
// row is rotated twice, for the maximum and for the codes; without the rotation
// 26 us); 1048 tokens 11.7 us (7.3 without); 256 tokens of a decode step 3 to 4 us.
#include <type_traits>

#include "fp8_common.cuh"

namespace mvb {

struct Fp8WriteArgs {
  const void* q;  // nullptr: no query rows
  int64_t q_s0, q_s1;
  void* q_out;
  int64_t qo_s0, qo_s1;
  const void* k;
  int64_t k_s0, k_s1;
  void* k_out;  // optional rotated keys [T, KH, D] contiguous
  const void* v;
  int64_t v_s0, v_s1;
  const int64_t* pos;  // nullptr: no rotation
  const void* cos;
  const void* sin;
  int64_t table_rows;
  uint8_t* kc;
  uint8_t* vc;
  float* scale;  // [num_blocks, KH, 2]
  const int64_t* slots;
  int* writer;  // [num_blocks * block_size], or nullptr: scan
  int num_tokens, num_heads, num_kv_heads, block_size, num_blocks;
  int* err;
};

namespace {

constexpr int kFp8ScanTokens = 2048;
constexpr int kFp8WriteThreads = 128;

// x c + y s, y the signed partner.  With 16-bit tables the product of two 16-bit
// floats is exact, and this is the exact rotation rounded once.
__device__ __forceinline__ float rope(float x, float c, float y, float s) {
  return __fmaf_rn(x, c, __fmul_rn(y, s));
}
// The same rounded once for float32 tables: the products and the sum with their
// rounding errors (exact by fma and by Knuth's two-sum), added back at the end.
__device__ __forceinline__ float rope_exact(float x, float c, float y, float s) {
  const float p1 = __fmul_rn(x, c), e1 = __fmaf_rn(x, c, -p1);
  const float p2 = __fmul_rn(y, s), e2 = __fmaf_rn(y, s, -p2);
  const float t = __fadd_rn(p1, p2);
  if (!(fabsf(t) < INFINITY)) return t;  // (the errors of infinities are NaN)
  const float b = __fsub_rn(t, p1);
  const float e3 = __fadd_rn(__fsub_rn(p1, __fsub_rn(t, b)), __fsub_rn(p2, b));
  return __fadd_rn(t, __fadd_rn(e3, __fadd_rn(e1, e2)));
}

// 4 consecutive elements as floats.
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&f)[4]) {
  if constexpr (sizeof(T) == 2) {
    const uint2 r = __ldg(reinterpret_cast<const uint2*>(p));
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_f32<T>(e[i]);
  } else {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
  }
}
// The token's slot if the token is written at all, else -1.
template <bool ROT>
__device__ __forceinline__ int64_t live_slot(const Fp8WriteArgs& a, int64_t total_slots, int t) {
  int64_t s = __ldg(a.slots + t);
  if (s >= total_slots) s = -1;
  if constexpr (ROT) {
    const int64_t p = __ldg(a.pos + t);
    if (p < 0 || p >= a.table_rows) s = -1;
  }
  return s < 0 ? -1 : s;
}

// What of token t only the device can see to be wrong.
template <bool ROT>
__device__ __forceinline__ void flag_token(const Fp8WriteArgs& a, int64_t total_slots, int t) {
  const int64_t raw = __ldg(a.slots + t);
  int bad = raw < -1 || raw >= total_slots ? MVB_DEV_SLOT_RANGE : 0;
  if constexpr (ROT) {
    const int64_t p = __ldg(a.pos + t);
    if (p < 0 || p >= a.table_rows) bad |= MVB_DEV_POSITION;
  }
  if (bad) atomicOr(a.err, bad);
}

template <bool ROT>
__global__ void __launch_bounds__(256) fp8_writer_kernel(const Fp8WriteArgs a) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.num_tokens) return;
  const int64_t s = live_slot<ROT>(a, (int64_t)a.num_blocks * a.block_size, t);
  if (s >= 0) a.writer[s] = t;
}


// Query rows, and key rows where the caller wants them: CTA `cta` of them, HPT
// rows of one token per thread.
template <typename T, typename TAB, int D, int HPT>
__device__ __forceinline__ void rotate_rows(const Fp8WriteArgs& a, int cta) {
  constexpr int LPR = D / 16;
  const int H = a.num_heads, rows = H + (a.k_out != nullptr ? a.num_kv_heads : 0);
  const int groups = (rows + HPT - 1) / HPT, d0 = (threadIdx.x % LPR) * 8;
  const int64_t tg = (int64_t)cta * (kFp8WriteThreads / LPR) + threadIdx.x / LPR;
  if (tg >= (int64_t)a.num_tokens * groups) return;
  const int t = (int)(tg / groups), r0 = (int)(tg - (int64_t)t * groups) * HPT;
  uint4 raw[HPT][2];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int r = min(r0 + i, rows - 1);
    const T* x = (r < H ? static_cast<const T*>(a.q) + (int64_t)t * a.q_s0 + (int64_t)r * a.q_s1
                        : static_cast<const T*>(a.k) + (int64_t)t * a.k_s0 + (int64_t)(r - H) * a.k_s1) + d0;
    // (plain loads: query_out may be query)
    raw[i][0] = *reinterpret_cast<const uint4*>(x);
    raw[i][1] = *reinterpret_cast<const uint4*>(x + D / 2);
  }
  const int64_t at = __ldg(a.pos + t);
  if (at < 0 || at >= a.table_rows) return;
  const TAB *cs = static_cast<const TAB*>(a.cos) + at * D + d0, *sn = static_cast<const TAB*>(a.sin) + at * D + d0;
#pragma unroll
  for (int half = 0; half < 2; ++half) {  // four columns of each half at a time
    float cl[4], ch[4], sl[4], sh[4];
    load4<TAB>(cs + 4 * half, cl);
    load4<TAB>(cs + D / 2 + 4 * half, ch);
    load4<TAB>(sn + 4 * half, sl);
    load4<TAB>(sn + D / 2 + 4 * half, sh);
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
      T *x = reinterpret_cast<T*>(&raw[i][0]) + 4 * half, *y = reinterpret_cast<T*>(&raw[i][1]) + 4 * half;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float u = to_f32<T>(x[k]), v = to_f32<T>(y[k]);
        x[k] = from_f32<T>(rope(u, cl[k], -v, sl[k]));
        y[k] = from_f32<T>(rope(v, ch[k], u, sh[k]));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int r = r0 + i;
    if (r >= rows) break;
    T* dst = (r < H ? static_cast<T*>(a.q_out) + (int64_t)t * a.qo_s0 + (int64_t)r * a.qo_s1
                    : static_cast<T*>(a.k_out) + ((int64_t)t * a.num_kv_heads + (r - H)) * D) + d0;
    *reinterpret_cast<uint4*>(dst) = raw[i][0];
    *reinterpret_cast<uint4*>(dst + D / 2) = raw[i][1];
  }
}

// One block's rows: the call's token at each of its slots is in map (-1: none).
template <typename T, typename TAB, int D, bool ROT>
__device__ __forceinline__ void write_block(const Fp8WriteArgs& a, const int* map, int64_t b0) {
  constexpr int LPR = D / 16, RPP = 32 / LPR, NWARP = kFp8WriteThreads / 32, NP = 16 / RPP;  // NP: passes at once
  const int KH = a.num_kv_heads, BS = a.block_size, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % LPR, place = lane / LPR, d0 = sub * 8;
  int rows = 0, only = 0;  // rows of the call, the last of them
  for (int r = lane; r < BS; r += 32)
    if (map[r] >= 0) {
      ++rows;
      only = r;
    }
  rows = __reduce_add_sync(0xffffffffu, rows);
  only = __reduce_max_sync(0xffffffffu, only);
  const bool single = rows == 1;  // each place of a warp has a (KV head, keys / values) of its own
  const int items = 2 * KH, per = single ? RPP : 1;
  for (int i0 = warp * per; i0 < items; i0 += NWARP * per) {
    const int it = single ? i0 + place : i0;
    const bool live = it < items;
    const int which = it < KH ? 0 : 1, kvh = live ? it - which * KH : 0;  // (keys, which are rotated, first)
    const int64_t bh = (b0 / BS) * KH + kvh;
    float* sp = a.scale + bh * 2 + which;
    const float old = map[0] >= 0 ? 0.f : *sp;
    uint8_t* codes = (which ? a.vc : a.kc) + bh * BS * D;
    const T* src = static_cast<const T*>(which ? a.v : a.k);
    const int64_t s0 = which ? a.v_s0 : a.k_s0;
    src += (int64_t)kvh * (which ? a.v_s1 : a.k_s1) + d0;
    // rows r0 + p RPP + place (or the only one) and their table rows
    uint4 raw[NP][2];
    int at[NP], pos[NP];
    auto load_rows = [&](int r0) {
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int r = single ? (p == 0 ? only : BS) : r0 + p * RPP + place;
        const int u = r < BS && live ? map[r] : -1;
        at[p] = u >= 0 ? r : -1;
        if (u < 0) continue;
        raw[p][0] = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)u * s0));
        raw[p][1] = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)u * s0 + D / 2));
        if (ROT && which == 0) pos[p] = (int)__ldg(a.pos + u);
      }
    };
    // pass p's row as float32, rotated: four columns of the lower and of the upper half at a time (rotated again where
    // it is coded: sixteen float32 values a row in registers spilled)
    auto row = [&](int p, auto exact, auto use) {
      const T *x = reinterpret_cast<const T*>(&raw[p][0]), *y = reinterpret_cast<const T*>(&raw[p][1]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = to_f32<T>(x[4 * half + i]);
          hi[i] = to_f32<T>(y[4 * half + i]);
        }
        if (ROT && which == 0) {
          const int64_t o = (int64_t)pos[p] * D + d0 + 4 * half;
          const TAB *cs = static_cast<const TAB*>(a.cos) + o, *sn = static_cast<const TAB*>(a.sin) + o;
          float cl[4], ch[4], sl[4], sh[4];
          load4<TAB>(cs, cl);
          load4<TAB>(cs + D / 2, ch);
          load4<TAB>(sn, sl);
          load4<TAB>(sn + D / 2, sh);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float u = lo[i], v = hi[i];
            if constexpr (decltype(exact)::value) {
              lo[i] = rope_exact(u, cl[i], -v, sl[i]);
              hi[i] = rope_exact(v, ch[i], u, sh[i]);
            } else {
              lo[i] = rope(u, cl[i], -v, sl[i]);
              hi[i] = rope(v, ch[i], u, sh[i]);
            }
          }
        }
        use(half, lo, hi);
      }
    };
    // the largest finite magnitude of this (KV head, keys / values)
    auto largest = [&](auto exact) {
      float amax = 0.f;
      for (int r0 = 0; r0 < BS; r0 += NP * RPP) {
        if (!decltype(exact)::value || BS > NP * RPP) load_rows(r0);  // (else they are still at hand)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          if (at[p] < 0) continue;
          row(p, exact, [&](int, const float (&lo)[4], const float (&hi)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = fabsf(lo[i]), y = fabsf(hi[i]);
              amax = fmaxf(amax, fmaxf(x < INFINITY ? x : 0.f, y < INFINITY ? y : 0.f));
            }
          });
        }
        if (single) break;
      }
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (!single) {
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      }
      return amax;
    };
    float amax = largest(std::false_type());
    if constexpr (ROT && sizeof(TAB) == 4) {
      // mantissa within 4 ulps of 1.75 (448 = 1.75 * 2^8)
      const bool border = (__float_as_uint(amax) & 0x7fffffu) - (0x600000u - 4u) <= 8u;
      if (__any_sync(0xffffffffu, border)) amax = largest(std::true_type());
    }
    const float base = old > 0.f && old < INFINITY ? old : 0.f;  // not a scale yet (or never): nothing to keep
    const float s = fmaxf(base, fp8_scale_for(amax));
    if (live && base > 0.f && s > base) {  // the scale has grown: the rows already there, 16 codes a lane
      const float ratio = __fdiv_rn(base, s);
#pragma unroll 4
      for (int r = single ? 0 : place; r < BS; r += single ? 1 : RPP) {
        if (map[r] >= 0) continue;
        uint4* p = reinterpret_cast<uint4*>(codes + (int64_t)r * D) + sub;
        uint4 w = *p;
        uint32_t* e = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t l, h;
          e4m3x4_to_f16(e[i], l, h);
          const float2 x = __half22float2(*reinterpret_cast<__half2*>(&l));
          const float2 y = __half22float2(*reinterpret_cast<__half2*>(&h));
          e[i] = f32x4_to_e4m3(x.x * ratio, x.y * ratio, y.x * ratio, y.y * ratio);
        }
        *p = w;
      }
    }
    const float inv = __frcp_rn(s);
    for (int r0 = 0; r0 < BS; r0 += NP * RPP) {
      if (!single && BS > NP * RPP) load_rows(r0);  // (else they are still at hand)
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        if (at[p] < 0) continue;
        uint2 l, h;
        row(p, std::bool_constant<ROT && sizeof(TAB) == 4>(), [&](int half, const float (&lo)[4], const float (&hi)[4]) {
          (half ? l.y : l.x) = f32x4_to_e4m3(lo[0] * inv, lo[1] * inv, lo[2] * inv, lo[3] * inv);
          (half ? h.y : h.x) = f32x4_to_e4m3(hi[0] * inv, hi[1] * inv, hi[2] * inv, hi[3] * inv);
        });
        uint8_t* to = codes + (int64_t)at[p] * D + d0;
        *reinterpret_cast<uint2*>(to) = l;
        *reinterpret_cast<uint2*>(to + D / 2) = h;
      }
      if (single) break;
    }
    __syncwarp();  // all lanes have read the old scale
    if (live && sub == 0 && (single || place == 0)) *sp = s;
  }
}

// Up to kFp8ScanTokens tokens: CTA t < num_tokens takes token t's block if the token is its leader, the CTAs behind
// them rotate the query rows.
template <typename T, typename TAB, int D, bool ROT>
__global__ void __launch_bounds__(kFp8WriteThreads, 4) fp8_write_kernel(const Fp8WriteArgs a) {
  extern __shared__ int map[];  // [block_size]
  grid_dependency_wait();
  grid_launch_dependents();
  if constexpr (ROT) {
    if ((int)blockIdx.x >= a.num_tokens) {
      rotate_rows<T, TAB, D, 2>(a, (int)blockIdx.x - a.num_tokens);
      return;
    }
  }
  const int t = blockIdx.x, tid = threadIdx.x, BS = a.block_size;
  const int64_t total_slots = (int64_t)a.num_blocks * BS;
  const int64_t slot = live_slot<ROT>(a, total_slots, t);
  const int64_t b0 = slot & ~(int64_t)(BS - 1);  // first slot of the block (BS is a power of two)
  const int off = (int)(slot - b0);
  if (tid == 0) flag_token<ROT>(a, total_slots, t);
  if (slot < 0) return;  // the same for all threads of the CTA
  for (int i = tid; i < BS; i += kFp8WriteThreads) map[i] = -1;
  __syncthreads();
  for (int u = tid; u < a.num_tokens; u += kFp8WriteThreads) {
    const int64_t s = live_slot<ROT>(a, total_slots, u);
    // two tokens of one slot: the later one is written, and the call is flagged
    if (s >= 0 && (s & ~(int64_t)(BS - 1)) == b0 && atomicMax(map + (s - b0), u) >= 0)
      atomicOr(a.err, MVB_DEV_DUP_SLOT);
  }
  __syncthreads();
  bool other = map[off] != t;  // some lower slot of the block is written, or this slot by another token
  for (int i = tid; i < off; i += kFp8WriteThreads) other |= map[i] >= 0;
  if (__syncthreads_or(other)) return;
  write_block<T, TAB, D, ROT>(a, map, b0);
}

// More tokens, behind fp8_writer_kernel: kFp8Chunk tokens a CTA, the query rows' CTAs behind them.
constexpr int kFp8Chunk = 8;
template <typename T, typename TAB, int D, bool ROT>
__global__ void __launch_bounds__(kFp8WriteThreads, 4) fp8_write_many_kernel(const Fp8WriteArgs a, int kv_ctas) {
  extern __shared__ int map[];  // [block_size]
  __shared__ int64_t slots[kFp8Chunk];  // -1: not a leader
  grid_dependency_wait();
  grid_launch_dependents();
  if constexpr (ROT) {
    if ((int)blockIdx.x >= kv_ctas) {
      rotate_rows<T, TAB, D, 4>(a, (int)blockIdx.x - kv_ctas);
      return;
    }
  }
  const int tid = threadIdx.x, BS = a.block_size;
  const int64_t total_slots = (int64_t)a.num_blocks * BS;
  if (tid < kFp8Chunk) {
    const int t = blockIdx.x * kFp8Chunk + tid;
    int64_t slot = -1;
    if (t < a.num_tokens) {
      flag_token<ROT>(a, total_slots, t);
      slot = live_slot<ROT>(a, total_slots, t);
      if (slot >= 0) {
        // this slot's entry is some token's of this call: if another's, that one wrote it last
        const bool dup = __ldcg(a.writer + slot) != t;
        if (dup) atomicOr(a.err, MVB_DEV_DUP_SLOT);
        // a chunk's next token: its left neighbour writes the slot before it
        if (dup || ((slot & (BS - 1)) != 0 && t > 0 && live_slot<ROT>(a, total_slots, t - 1) == slot - 1)) slot = -1;
      }
    }
    slots[tid] = slot;
  }
  __syncthreads();
  for (int k = 0; k < kFp8Chunk; ++k) {
    const int64_t slot = slots[k];
    if (slot < 0) continue;  // the same for all threads of the CTA
    const int64_t b0 = slot & ~(int64_t)(BS - 1);
    bool other = false;  // some lower slot of the block is written
    for (int i = tid; i < BS; i += kFp8WriteThreads) {
      const int w = __ldcg(a.writer + b0 + i);
      const bool ok = w >= 0 && w < a.num_tokens && live_slot<ROT>(a, total_slots, w) == b0 + i;
      map[i] = ok ? w : -1;
      other |= ok && b0 + i < slot;
    }
    if (!__syncthreads_or(other)) write_block<T, TAB, D, ROT>(a, map, b0);
    __syncthreads();
  }
}

template <typename T, typename TAB, int D, bool ROT>
int launch_write(const Fp8WriteArgs& a, cudaStream_t stream) {
  const int smem = a.block_size * 4;
  const int rows = a.num_heads + (a.k_out != nullptr ? a.num_kv_heads : 0);
  auto rotate_ctas = [&](int heads) -> int64_t {
    const int64_t items = (int64_t)a.num_tokens * ((rows + heads - 1) / heads) * (D / 16);
    return ROT ? (items + kFp8WriteThreads - 1) / kFp8WriteThreads : 0;
  };
  if (a.num_tokens + rotate_ctas(2) >= ((int64_t)1 << 31)) return MVB_ERR_INVALID_ARG;
  if (a.writer == nullptr) {
    auto kern = fp8_write_kernel<T, TAB, D, ROT>;
    if (ensure_kernel_attrs(kern, smem) != cudaSuccess) return MVB_ERR_CUDA;
    return launch_pdl(kern, dim3((unsigned)(a.num_tokens + rotate_ctas(2))), dim3(kFp8WriteThreads), smem, stream, a) ==
                   cudaSuccess
               ? MVB_OK
               : MVB_ERR_CUDA;
  }
  auto first = fp8_writer_kernel<ROT>;
  auto kern = fp8_write_many_kernel<T, TAB, D, ROT>;
  if (ensure_kernel_attrs(first, 0) != cudaSuccess || ensure_kernel_attrs(kern, smem) != cudaSuccess) return MVB_ERR_CUDA;
  if (launch_pdl(first, dim3((a.num_tokens + 255) / 256), dim3(256), 0, stream, a) != cudaSuccess) return MVB_ERR_CUDA;
  const int kv_ctas = (a.num_tokens + kFp8Chunk - 1) / kFp8Chunk;
  return launch_pdl(kern, dim3((unsigned)(kv_ctas + rotate_ctas(4))), dim3(kFp8WriteThreads), smem, stream, a, kv_ctas) ==
                 cudaSuccess
             ? MVB_OK
             : MVB_ERR_CUDA;
}

template <typename T>
int launch_write_t(const Fp8WriteArgs& a, int head_dim, bool f32_tables, cudaStream_t stream) {
  if (a.pos == nullptr)
    return head_dim == 64 ? launch_write<T, T, 64, false>(a, stream) : launch_write<T, T, 128, false>(a, stream);
  if (f32_tables)
    return head_dim == 64 ? launch_write<T, float, 64, true>(a, stream) : launch_write<T, float, 128, true>(a, stream);
  return head_dim == 64 ? launch_write<T, T, 64, true>(a, stream) : launch_write<T, T, 128, true>(a, stream);
}

int write_fp8(Fp8WriteArgs a, int head_dim, int dtype, int table_dtype, void* workspace, int64_t workspace_bytes,
              void* stream) {
  if (dtype != MVB_DTYPE_F16 && dtype != MVB_DTYPE_BF16) return MVB_ERR_DTYPE;
  if (a.pos != nullptr && table_dtype != dtype && table_dtype != MVB_DTYPE_F32) return MVB_ERR_DTYPE;
  if (head_dim != 64 && head_dim != 128) return MVB_ERR_HEAD_DIM;
  if (a.block_size < kFp8MinBlock || a.block_size > kFp8MaxBlock || (a.block_size & (a.block_size - 1)) != 0)
    return MVB_ERR_BLOCK_SIZE;
  if (a.num_tokens < 0 || a.num_kv_heads <= 0 || a.num_blocks <= 0) return MVB_ERR_INVALID_ARG;
  if (a.num_tokens == 0) return MVB_OK;
  if (!a.k || !a.v || !a.kc || !a.vc || !a.scale || !a.slots || !a.err) return MVB_ERR_INVALID_ARG;
  auto al = [](const void* p, int64_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  auto al_s = [](int64_t s) { return s % 8 == 0; };  // 16-byte vectors of 16-bit elements
  if (!al(a.k, 16) || !al(a.v, 16) || !al(a.kc, 16) || !al(a.vc, 16) || !al(a.scale, 4) || !al_s(a.k_s0) ||
      !al_s(a.k_s1) || !al_s(a.v_s0) || !al_s(a.v_s1) || !al(a.k_out, 16))
    return MVB_ERR_ALIGNMENT;
  if (a.pos != nullptr && a.table_rows >= ((int64_t)1 << 31)) return MVB_ERR_INVALID_ARG;
  if (a.pos != nullptr &&
      (!al(a.q, 16) || !al(a.q_out, 16) || !al(a.cos, 16) || !al(a.sin, 16) || !al_s(a.q_s0) || !al_s(a.q_s1) ||
       !al_s(a.qo_s0) || !al_s(a.qo_s1)))
    return MVB_ERR_ALIGNMENT;
  a.writer = nullptr;
  if (a.num_tokens > kFp8ScanTokens) {
    if (workspace == nullptr || workspace_bytes < (int64_t)a.num_blocks * a.block_size * 4 || !al(workspace, 4))
      return MVB_ERR_WORKSPACE;
    a.writer = static_cast<int*>(workspace);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f32_tables = table_dtype == MVB_DTYPE_F32;
  return dtype == MVB_DTYPE_BF16 ? launch_write_t<__nv_bfloat16>(a, head_dim, f32_tables, s)
                                 : launch_write_t<__half>(a, head_dim, f32_tables, s);
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int mvb_kv_cache_write_fp8_workspace(int32_t num_tokens, int32_t num_blocks, int32_t block_size,
                                                int64_t* bytes_out) {
  if (num_tokens < 0 || num_blocks <= 0 || block_size <= 0 || !bytes_out) return MVB_ERR_INVALID_ARG;
  *bytes_out = num_tokens <= kFp8ScanTokens ? 0 : (int64_t)num_blocks * block_size * 4;
  return MVB_OK;
}

extern "C" int mvb_kv_cache_write_fp8(const void* key, int64_t k_stride_token, int64_t k_stride_head,
                                      const void* value, int64_t v_stride_token, int64_t v_stride_head,
                                      void* key_cache, void* value_cache, float* kv_scale,
                                      const int64_t* slot_mapping, int32_t num_tokens, int32_t num_kv_heads,
                                      int32_t head_dim, int32_t block_size, int32_t num_blocks, int32_t dtype,
                                      void* workspace, int64_t workspace_bytes, int32_t* error_flags, void* stream) {
  mvb::NvtxRange nvtx_range("mvb_kv_cache_write_fp8");
  Fp8WriteArgs a = {};
  a.k = key;
  a.k_s0 = k_stride_token;
  a.k_s1 = k_stride_head;
  a.v = value;
  a.v_s0 = v_stride_token;
  a.v_s1 = v_stride_head;
  a.kc = static_cast<uint8_t*>(key_cache);
  a.vc = static_cast<uint8_t*>(value_cache);
  a.scale = kv_scale;
  a.slots = slot_mapping;
  a.num_tokens = num_tokens;
  a.num_kv_heads = num_kv_heads;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.err = error_flags;
  return write_fp8(a, head_dim, dtype, dtype, workspace, workspace_bytes, stream);
}

extern "C" int mvb_rope_kv_cache_write_fp8(
    const void* query, int64_t q_stride_token, int64_t q_stride_head, void* query_out, int64_t qo_stride_token,
    int64_t qo_stride_head, const void* key, int64_t k_stride_token, int64_t k_stride_head, const void* value,
    int64_t v_stride_token, int64_t v_stride_head, const int64_t* positions, const void* cos_table,
    const void* sin_table, int64_t table_rows, int32_t table_dtype, void* key_cache, void* value_cache,
    float* kv_scale, const int64_t* slot_mapping, void* key_out, int32_t num_tokens, int32_t num_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t num_blocks, int32_t dtype, void* workspace,
    int64_t workspace_bytes, int32_t* error_flags, void* stream) {
  mvb::NvtxRange nvtx_range("mvb_rope_kv_cache_write_fp8");
  if (num_heads <= 0 || table_rows <= 0) return MVB_ERR_INVALID_ARG;
  if (num_tokens > 0 && (!query || !query_out || !positions || !cos_table || !sin_table)) return MVB_ERR_INVALID_ARG;
  Fp8WriteArgs a = {};
  a.q = query;
  a.q_s0 = q_stride_token;
  a.q_s1 = q_stride_head;
  a.q_out = query_out;
  a.qo_s0 = qo_stride_token;
  a.qo_s1 = qo_stride_head;
  a.k = key;
  a.k_s0 = k_stride_token;
  a.k_s1 = k_stride_head;
  a.k_out = key_out;
  a.v = value;
  a.v_s0 = v_stride_token;
  a.v_s1 = v_stride_head;
  a.pos = positions;
  a.cos = cos_table;
  a.sin = sin_table;
  a.table_rows = table_rows;
  a.kc = static_cast<uint8_t*>(key_cache);
  a.vc = static_cast<uint8_t*>(value_cache);
  a.scale = kv_scale;
  a.slots = slot_mapping;
  a.num_tokens = num_tokens;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.err = error_flags;
  return write_fp8(a, head_dim, dtype, table_dtype, workspace, workspace_bytes, stream);
}
