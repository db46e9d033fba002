// mvb_paged_decode_fp8: attention of one query token per sequence over an
// 8-bit paged cache with a scale per (block, KV head):
//   out[s, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j - max),
//   k_j = code * kv_scale[block(j), kvh, 0],  v_j = code * kv_scale[block(j), kvh, 1].
//
// Math of one 16-token tile (one warp).  The tile's tokens are the rows of the
// tensor-core product and the KV head's query heads its 8 columns (a head
// group; 16 heads are two column blocks), so 7 heads waste one column where
// heads as rows would waste 9 of 16:
//   S^T[16 tokens, 8 heads] = K_codes Q^T,   O^T[D, 8 heads] = V_codes^T P^T.
// * A tile is 16 D contiguous bytes of K and of V.  Each warp copies its tiles
//   into a ring of its own (Fp8Geo::STAGES tiles, TMA, one mbarrier a stage) and
//   turns codes into f16 (exact) in registers: the sum over D may run in any
//   order, so a lane's 16 contiguous bytes of a K row serve four k-steps, and its
//   8 (D = 64) or 16 contiguous bytes of four V rows are D/8 rows of O^T.  The
//   same ring filled by cp.async stayed at 5.1 TB/s with no arithmetic at all.
// * The query enters as f16, each head's row times a power of two that brings
//   its largest element into [1, 2): exact for f16 queries and for bf16 ones but
//   for elements below 2^-14 of the row's largest, which lose bits under 2^-24
//   of it.
// * All tokens of a tile lie in one block, so the key scale is one factor of the
//   tile's logits.  The value scale v joins the exponent: P = p v / R, with the
//   sum of p undone per tile, O in units of R, a power of two: the first tile's
//   scale, moved (O with it) when a scale passes 2^7 R.  The exponent takes v / R
//   down to 2^-4, where P's f16 still has 10 bits for p >= 2^-10; the rest of a
//   smaller scale goes into the f16 codes (exact to 2^-15 R).
// * P enters as f16 (11 bits; the output has 8 or 11), against a maximum m of
//   earlier tiles; m is taken anew only when a lane's P add up to more than 2^14
//   (once a tile), so a tile needs no reduction across lanes, only a vote.
// * With a factor on every output of a tile and a maximum per tile, one tile at a
//   time, it took 204 instructions per tile of head_dim 64 and was bound by them.
//
// Work split: the tiles of all (sequence, KV head, head group) units in order
// are one stream, cut into equal ranges, one per warp of a grid of at most one
// CTA per SM (or each unit is a CTA's own: see kFp8WholeTiles).  A unit inside a warp's range is written at once.  The pieces of
// units cut between the warps of a CTA are merged in shared memory; only a unit
// cut between two CTAs leaves partial states in global memory, which
// fp8_decode_merge_kernel joins in CTA order.  The workspace holds nothing from
// one call to the next and needs no initialisation.
// Bound: memory (1 byte per element; 28 operations per byte at 7 heads), short
// sequences by the launches and the first loads.  Measured: 256 sequences of 32/8
// heads of 128, 817 MB: 157 us, 5.2 TB/s (141 us, 5.8 TB/s in a graph); 32 x 32768
// tokens of 14/2 heads of 64, 270 MB: 60 us, 4.5 TB/s; 256 x 2048: 29 us, 16 of them the
// stream (4.7 TB/s), the rest prologue and merges.
#include <cudaTypedefs.h>

#include <algorithm>
#include <type_traits>

#include "fp8_common.cuh"

namespace mvb {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn();  // capi.cu

struct Fp8DecodeArgs {
  const void* q;
  int64_t q_s0, q_s1;
  const uint8_t* kc;
  const uint8_t* vc;
  const float2* scale;  // [num_blocks, KH] (key, value)
  const int64_t* bt;
  int64_t bt_s0;
  int max_blocks;
  const int* kv_len;
  void* out;
  int64_t o_s0, o_s1;
  int num_seqs, num_heads, num_kv_heads, G, head_groups, block_shift, num_blocks;
  float scale_log2;
  int whole;    // a CTA per unit, each with all of its tiles
  float* part;  // [grid][2][16 * (D + 2)] partial states of units cut between CTAs: O, then (m, l)
  int4* desc;   // [grid][2] {unit (-1: none), sequence, first head, heads}; slot 0: the unit began earlier
  int* err;
};

namespace {

constexpr int kFp8Tile = 16;
constexpr int kFp8DecodeMaxSeqs = 6144;  // the tile prefix lies in shared memory
// log2 of (value scale / reference) that P takes up.
constexpr float kMinValueExp = -4.f, kMaxValueExp = 7.f;
// A warp gets at least this many tiles where the batch has few.
constexpr int kFp8MinTiles = 2;
// A CTA takes a unit of its own, and nothing is left to merge in a second launch, where
// there are SMs for all units, a unit has at most kFp8WholeTiles tiles per warp, and
// that is at most kFp8WholeMore more than an equal share of the stream would be: a
// tile costs a warp about 0.7 us, the merge 3 to 4.  Shared and whole (us): 1 x 1000,
// 14/2 heads of 64: 10.6 and 9.4; 64 x 1000: 14.7 and 10.7; 64 x 2000: 18.1 and 13.7;
// 16 x 1500, 32/8 of 128: 19.0 and 15.4; but 1 x 2000: 10.8 and 12.3, 1 x 4000: 11.6
// and 18.5.  The first limit is for tables wider than most sequences need.
constexpr int kFp8WholeTiles = 8, kFp8WholeMore = 4;

// Geometry by head_dim and column blocks: warps per CTA and tiles in a warp's
// ring.  The rings, a piece per warp and the prefix of the largest batch fill
// shared memory.
template <int D, int NG> struct Fp8Geo;
template <> struct Fp8Geo<64, 1> { static constexpr int NW = 16, STAGES = 5; };
template <> struct Fp8Geo<64, 2> { static constexpr int NW = 12, STAGES = 5; };
template <> struct Fp8Geo<128, 1> { static constexpr int NW = 12, STAGES = 3; };
template <> struct Fp8Geo<128, 2> { static constexpr int NW = 8, STAGES = 4; };

template <int D, int NG> struct Fp8Smem {
  static constexpr int NW = Fp8Geo<D, NG>::NW, TILE = 2 * 16 * D;  // K, then V
  static constexpr int PIECE = 8 * NG * (D + 2) * 4;  // bytes of one partial state: O [8 NG][D], then (m, l) [8 NG]
  static constexpr int RING = 0, PARTS = RING + NW * Fp8Geo<D, NG>::STAGES * TILE, IDS = PARTS + NW * PIECE;
  static constexpr int BARS = IDS + NW * 2 * 16, PRE = BARS + NW * Fp8Geo<D, NG>::STAGES * 8;
  // (the prefix gives way to the list of cut units at the end; 1024 for the alignment)
  static constexpr int bytes(int num_seqs) { return PRE + (num_seqs < 64 ? 64 : num_seqs + 1) * 4 + 1024; }
  static_assert(2 * (NW + 1) <= 64, "the list fits");
  static_assert(Fp8Geo<D, NG>::STAGES * TILE >= PIECE, "a warp's second piece lies in its ring");
  static_assert(bytes(kFp8DecodeMaxSeqs) + 128 <= 227 * 1024, "shared memory of one CTA");
};

// Byte offset of 16-byte chunk c of token r of a tile as the TMA load leaves it: rows of 128 bytes (two tokens at
// D = 64: boxes of 64-byte rows stayed at 4.6 TB/s), chunks swizzled by the row.
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  const int b = r * D + c * 16, row = b >> 7;
  return (uint32_t)(row * 128 + ((b & 127) ^ ((row & 7) << 4)));
}
// The same chunk 8 tokens on.
template <int D>
__device__ __forceinline__ uint32_t on8(uint32_t at) { return D == 64 ? (at ^ 64) + 512 : at + 1024; }
// Token of row r (0-7, and 8 more) of a tile's product: an order in which the chunks that eight lanes (K, and V at
// D = 128) or sixteen lanes (V at D = 64, 8 bytes each) read at once lie in different banks.
template <int D>
__device__ __forceinline__ int token_of(int r) { return D == 64 ? r ^ (r >> 1 & 1) : r ^ ((r & 1) << 2); }
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
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
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One unit of the stream.
struct Unit {
  int start, end;  // its tiles [start, end) of the stream
  int seq, k;      // sequence, unit of the sequence
};

template <typename T, int D, int NG>
__global__ void __launch_bounds__(Fp8Geo<D, NG>::NW * 32, 1)
fp8_decode_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                  const Fp8DecodeArgs a) {
  using Sm = Fp8Smem<D, NG>;
  constexpr int NW = Fp8Geo<D, NG>::NW, ST = Fp8Geo<D, NG>::STAGES;
  constexpr int HR = 8 * NG, MT = D / 16, KS = D / 16, KW = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int4* ids = reinterpret_cast<int4*>(smem + Sm::IDS);  // [NW][2] {unit, seq, k, ends in this CTA}
  int* pre = reinterpret_cast<int*>(smem + Sm::PRE);    // [Nd + 1] tile prefix
  __shared__ int sums[NW];
  // A warp's partial states: slot 0 of a unit that began before its range, slot 1 (in its ring, at the end) of one
  // that runs on.
  auto part_of = [&](int w, int slot) {
    return reinterpret_cast<float*>(smem + (slot == 0 ? Sm::PARTS + w * Sm::PIECE : Sm::RING + w * ST * Sm::TILE));
  };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int Nd = a.num_seqs, KHG = a.num_kv_heads * a.head_groups;
  T* const out = static_cast<T*>(a.out);
  if (tid == 0) {
    prefetch_tensormap(&tmk);
    prefetch_tensormap(&tmv);
  }
  grid_dependency_wait();
  grid_launch_dependents();

  // ---- tiles of every sequence (all its units) and their exclusive prefix ----
  {
    constexpr int NT = NW * 32;
    const int per = (Nd + NT - 1) / NT;
    const int i0 = min(Nd, tid * per), i1 = min(Nd, i0 + per);
    int mine = 0;
    for (int i = i0; i < i1; ++i) {
      const int c = __ldg(a.kv_len + i);
      const int bad = c < 1 ? MVB_DEV_KV_LEN
                      : ((int64_t)c + (1 << a.block_shift) - 1) >> a.block_shift > a.max_blocks ? MVB_DEV_TABLE_SHORT
                                                                                               : 0;
      const int n = bad ? 0 : ((c - 1) / kFp8Tile + 1) * KHG;
      pre[i] = n;
      mine += n;
      if (bad && blockIdx.x == 0) atomicOr(a.err, bad);
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sums[warp] = incl;
    if (tid < NW * 2) ids[tid] = make_int4(-1, 0, 0, 0);
    __syncthreads();
    int run = incl - mine, total = 0;
    for (int w = 0; w < NW; ++w) {
      if (w < warp) run += sums[w];
      total += sums[w];
    }
    for (int i = i0; i < i1; ++i) {
      const int n = pre[i];
      pre[i] = run;
      run += n;
    }
    if (tid == 0) pre[Nd] = total;
    __syncthreads();
  }
  // rows of sequences that cannot be served: zeros
  for (int i = blockIdx.x * NW + warp; i < Nd; i += gridDim.x * NW) {
    if (pre[i] != pre[i + 1]) continue;
    for (int e = lane; e < a.num_heads * D; e += 32)
      out[(int64_t)i * a.o_s0 + (int64_t)(e / D) * a.o_s1 + e % D] = from_f32<T>(0.f);
  }

  // this CTA's share of the stream, [base, base + T), or with others' all of it, and the first of its W warps there
  int base = 0, T_all = pre[Nd], ctas = gridDim.x, first = blockIdx.x * NW;
  if (a.whole) {
    const int seq = blockIdx.x / KHG;
    T_all = (pre[seq + 1] - pre[seq]) / KHG;
    base = pre[seq] + (blockIdx.x - seq * KHG) * T_all;
    ctas = 1;
    first = 0;
  }
  const int W = min(min(ctas, max(1, (T_all + NW * kFp8MinTiles - 1) / (NW * kFp8MinTiles))) * NW, max(T_all, 1));
  auto bound = [&](int w) { return base + (int)((int64_t)min(w, W) * T_all / W); };
  const int r0 = bound(first + warp), r1 = bound(first + warp + 1);
  const int c0 = bound(first), c1 = bound(first + NW);

  auto unit_at = [&](int tile) {
    int lo = 0, hi = Nd;  // pre[lo] <= tile < pre[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= tile)
        lo = mid;
      else
        hi = mid;
    }
    Unit u;
    u.seq = lo;
    const int n = (pre[lo + 1] - pre[lo]) / KHG;
    u.k = (tile - pre[lo]) / n;
    u.start = pre[lo] + u.k * n;
    u.end = u.start + n;
    return u;
  };
  const int BSm = (1 << a.block_shift) - 1, gshift = a.block_shift - 4;
  const uint64_t policy = l2_policy_evict_first();
  // Lane-wise: tile `tile` of the stream, numbered among the cache's 16-token groups; for a bad block id group 0,
  // which is read and not counted.
  auto find_tile = [&](int tile, bool& missing) {
    const Unit u = unit_at(tile);
    const int tok = (tile - u.start) * kFp8Tile;
    const int64_t b = __ldg(a.bt + (int64_t)u.seq * a.bt_s0 + (tok >> a.block_shift));
    if (b >= 0 && b < a.num_blocks)
      return ((uint32_t)((int)b * a.num_kv_heads + u.k / a.head_groups) << gshift) + ((uint32_t)(tok & BSm) >> 4);
    atomicOr(a.err, MVB_DEV_BLOCK_ID);
    missing = true;
    return 0u;
  };

  if (r0 < r1) {
    // 32 tiles' places and scales at a time, one per lane; the next 32 are fetched ahead
    uint32_t grp = 0, grp_n = 0;
    bool missing = false;
    if (r0 + lane < r1) grp = find_tile(r0 + lane, missing);
    const uint32_t ring = smem_u32(smem + Sm::RING + warp * ST * Sm::TILE);
    const uint32_t bars = smem_u32(smem + Sm::BARS + warp * ST * 8);
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < ST; ++i) mbar_init(bars + 8 * i, 1);
      fence_mbar_init();
    }
    __syncwarp();
    int put = 0;  // stage that is filled next
    // Start the copies of the tile `j` places into the current 32 (or the next 32's).
    auto issue = [&](int j) {
      const uint32_t g = __shfl_sync(0xffffffffu, j < 32 ? grp : grp_n, j & 31);
      if (lane == 0) {
        const uint32_t bar = bars + 8 * put, dst = ring + put * Sm::TILE;
        mbar_arrive_expect_tx(bar, Sm::TILE);
        tma_load_2d(dst, &tmk, 0, (int)(g * (D / 8)), bar, policy);
        tma_load_2d(dst + 16 * D, &tmv, 0, (int)(g * (D / 8)), bar, policy);
      }
      put = put + 1 == ST ? 0 : put + 1;
    };
    int next = r0;  // the tile that is started next
#pragma unroll
    for (int b = 0; b < ST; ++b)
      if (next < r1) {
        issue(b);
        ++next;
      }
    // what else the first step needs, all on its way at once: scales, lengths, queries, the next places
    auto scales_raw = [&](uint32_t group) {
      float2 x;
      asm volatile("ld.global.nc.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "l"(a.scale + (group >> gshift)));
      return x;
    };
    // a group's key scale and log2 of its value scale (exact for a power of two)
    auto scales = [&](float2 x) {
      const uint32_t bits = __float_as_uint(x.y);
      x.y = (bits & 0x7fffffu) == 0 && bits != 0 ? (float)((int)(bits >> 23) - 127) : log2f(x.y);
      return x;
    };
    float2 sc = scales_raw(grp), sc_n = make_float2(1.f, 1.f);
    Unit u = unit_at(r0);
    int h0 = 0, nh = 0, ctx = 0;
    uint4 qraw[NG][KW][2];
    auto load_q = [&]() {
      const int kvh = u.k / a.head_groups, hg = u.k - kvh * a.head_groups;
      h0 = kvh * a.G + hg * HR;
      nh = min(HR, a.G - hg * HR);
      asm volatile("ld.global.nc.s32 %0, [%1];" : "=r"(ctx) : "l"(a.kv_len + u.seq));
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const int h = 8 * n + g;
        const T* qp = static_cast<const T*>(a.q) + (int64_t)u.seq * a.q_s0 + (int64_t)(h0 + h) * a.q_s1 + 16 * t4;
#pragma unroll
        for (int c = 0; c < KW; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint4& r = qraw[n][c][i];
            r = make_uint4(0, 0, 0, 0);
            if (h < nh)
              asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                           : "l"(qp + 64 * c + 8 * i));
          }
      }
    };
    load_q();
    uint32_t bad = __ballot_sync(0xffffffffu, missing);  // places of the current 32 without a block
    missing = false;
    if (r0 + 32 + lane < r1) grp_n = find_tile(r0 + 32 + lane, missing);
    sc = scales(sc);

    int j = 0;           // the current tile's place in the current 32
    int get = 0;         // its stage, and that one's phase
    uint32_t phase = 0;
    bool late = false;   // a bounded wait ran out: what was read is not the cache
    uint32_t qf[NG][KS][2];
    float qs[NG][2];  // per column (heads 2t, 2t + 1): softmax scale, log2 e, the query row's power of two
    float o[NG][MT][4], m[NG][2], l[NG][2];
    float R = 0.f;       // log2 of the reference that O is in units of, once a tile has given it
    bool have_r = false;
    bool fresh = true;   // the unit has no maximum yet
    auto begin_unit = [&]() {
      R = 0.f;
      have_r = false;
      fresh = true;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float x[KW][16], amax = 0.f;
#pragma unroll
        for (int c = 0; c < KW; ++c) {
          const T* e = reinterpret_cast<const T*>(qraw[n][c]);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            x[c][i] = to_f32<T>(e[i]);
            const float y = fabsf(x[c][i]);
            amax = fmaxf(amax, y < INFINITY ? y : 0.f);
          }
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^-e with e = floor(log2 amax), kept where both 2^e and 2^-e are normal
        const int e = min(max((int)(__float_as_uint(amax) >> 23), 2), 252);
        const float down = __uint_as_float((uint32_t)(254 - e) << 23), up = __uint_as_float((uint32_t)e << 23);
#pragma unroll
        for (int c = 0; c < KW; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            qf[n][4 * c + k][0] = pack_h2(x[c][4 * k] * down, x[c][4 * k + 1] * down);
            qf[n][4 * c + k][1] = pack_h2(x[c][4 * k + 2] * down, x[c][4 * k + 3] * down);
          }
        // lane (g, t) holds head 8n + g's factor; its columns are heads 2t and 2t + 1
        qs[n][0] = a.scale_log2 * __shfl_sync(0xffffffffu, up, (2 * t4) * 4);
        qs[n][1] = a.scale_log2 * __shfl_sync(0xffffffffu, up, (2 * t4 + 1) * 4);
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      }
    };
    // The unit is finished in this range: written, or left as a piece.
    auto end_unit = [&]() {
      const bool whole = u.start >= r0 && u.end <= r1;
      const int slot = u.start < r0 ? 0 : 1;
      const float unit_of_o = fast_exp2(R);
      float* P = part_of(warp, slot);
      if (!whole && lane == 0) ids[warp * 2 + slot] = make_int4(u.start, u.seq, u.k, u.end <= c1 ? 1 : 0);
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float s = l[n][c];
          s += __shfl_xor_sync(0xffffffffu, s, 4);
          s += __shfl_xor_sync(0xffffffffu, s, 8);
          s += __shfl_xor_sync(0xffffffffu, s, 16);
          const int h = 8 * n + 2 * t4 + c;
          if (h >= nh) continue;
          // this lane's D / 8 contiguous dims of head h: element 2i + half of o[i][c + 2 half]
          if (whole) {
            const float inv = s == 0.f ? 0.f : unit_of_o / s;
            T* p = out + (int64_t)u.seq * a.o_s0 + (int64_t)(h0 + h) * a.o_s1 + (D / 8) * g;
            uint32_t w[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              T e[2] = {from_f32<T>(o[n][i][c] * inv), from_f32<T>(o[n][i][c + 2] * inv)};
              w[i] = *reinterpret_cast<uint32_t*>(e);
            }
#pragma unroll
            for (int i = 0; i < MT / 4; ++i)
              reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          } else {
            float* p = P + h * D + (D / 8) * g;
#pragma unroll
            for (int i = 0; i < MT / 2; ++i)
              *reinterpret_cast<float4*>(p + 4 * i) =
                  make_float4(o[n][2 * i][c] * unit_of_o, o[n][2 * i][c + 2] * unit_of_o,
                              o[n][2 * i + 1][c] * unit_of_o, o[n][2 * i + 1][c + 2] * unit_of_o);
            if (g == 0) *reinterpret_cast<float2*>(P + HR * D + 2 * h) = make_float2(m[n][c], s);
          }
        }
    };
    begin_unit();

    // rows g and g + 8 of K, and rows 2t, 2t + 1, 2t + 8, 2t + 9 of V, in a stage
    const int tok_g = token_of<D>(g);
    const uint32_t k_at = chunk_at<D>(tok_g, t4);  // (64 columns on, at D = 128: bit 6)
    uint32_t v_at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v_at[i] = KW == 1 ? chunk_at<D>(token_of<D>(2 * t4 + i), g >> 1) + 8 * (g & 1) : chunk_at<D>(token_of<D>(2 * t4 + i), g);
    // Tiles [tile, tile + NT) of one unit (their places j and on are in the current 32).
    auto attend = [&](int tile, auto count) {
      constexpr int NT = decltype(count)::value, WR = D / 32;  // WR: words of one V row in this lane
      __syncwarp();  // all lanes are done with the tiles before: their stages are free
#pragma unroll
      for (int b = 0; b < (D == 64 ? 2 : 1); ++b)
        if (next < r1 && next < tile + ST) {
          issue(j + next - tile);
          ++next;
        }
      uint32_t stage[NT];
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        if (!mbar_wait_bounded(bars + 8 * get, phase)) late = true;
        stage[b] = (uint32_t)(Sm::RING + (warp * ST + get) * Sm::TILE);
        if (++get == ST) {
          get = 0;
          phase ^= 1;
        }
      }
      float ks[NT], ve[NT], rest[NT];
      bool odd = !have_r;
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        ks[b] = __shfl_sync(0xffffffffu, sc.x, j + b);
        ve[b] = __shfl_sync(0xffffffffu, sc.y, j + b) - R;
        rest[b] = 1.f;
        odd |= !(fabsf(ve[b] - 0.5f * (kMinValueExp + kMaxValueExp)) <= 0.5f * (kMaxValueExp - kMinValueExp));
      }
      // the unit's last tile, or places without a block: some tokens do not count
      const bool edge = tile + NT >= u.end || (bad >> j & ((1u << NT) - 1)) != 0;
      int valid[NT];
#pragma unroll
      for (int b = 0; b < NT; ++b) valid[b] = (bad >> (j + b)) & 1 ? 0 : ctx - (tile + b - u.start) * kFp8Tile;
      if (odd) {  // value scales that R does not serve
#pragma unroll
        for (int b = 0; b < NT; ++b) {
          if ((ve[b] > kMaxValueExp || !have_r) && ve[b] > -INFINITY) {  // R moves, and O with it
            const float up = floorf(ve[b]), f = fast_exp2(-up);
            R += up;
#pragma unroll
            for (int i = 0; i < NT; ++i) ve[i] -= up;
            if (have_r) {
#pragma unroll
              for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[n][i][e] *= f;
            }
            have_r = true;
          }
        }
        odd = false;
#pragma unroll
        for (int b = 0; b < NT; ++b)
          if (ve[b] < kMinValueExp) {
            rest[b] = fast_exp2(ve[b] - kMinValueExp);
            ve[b] = kMinValueExp;
            odd = true;
          }
      }
      // S^T = K Q^T
      float s[NT][NG][4];
#pragma unroll
      for (int b = 0; b < NT; ++b) {
#pragma unroll
        for (int n = 0; n < NG; ++n) s[b][n][0] = s[b][n][1] = s[b][n][2] = s[b][n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < KW; ++c) {
          const uint4 x4 = *reinterpret_cast<const uint4*>(smem + stage[b] + (k_at ^ (c << 6))),
                      y4 = *reinterpret_cast<const uint4*>(smem + stage[b] + on8<D>(k_at ^ (c << 6)));
          const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_f16(x[k], a0, a2);
            e4m3x4_to_f16(y[k], a1, a3);
#pragma unroll
            for (int n = 0; n < NG; ++n) mma_f16(s[b][n], a0, a1, a2, a3, qf[n][4 * c + k][0], qf[n][4 * c + k][1]);
          }
        }
      }
      uint32_t v[NT][4 * WR];
#pragma unroll
      for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* p = smem + stage[b] + 16 * D + (i < 2 ? v_at[i] : on8<D>(v_at[i & 1]));
          if constexpr (KW == 1) {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            v[b][2 * i] = x.x, v[b][2 * i + 1] = x.y;
          } else {
            const uint4 x = *reinterpret_cast<const uint4*>(p);
            v[b][4 * i] = x.x, v[b][4 * i + 1] = x.y, v[b][4 * i + 2] = x.z, v[b][4 * i + 3] = x.w;
          }
        }
      // P against the maximum of earlier tiles, which is taken anew, once, where a lane's P add up to more than 2^14.
      // An exponent is a fused multiply-add: its product is not rounded, so it can lie half an ulp of m above the
      // maximum of the rounded ones (2^4 from |m| = 2^28 on).  Against a maximum just taken it is therefore the
      // difference of the rounded ones: 0 at the largest, nowhere above the tile's ve, whatever the logits' size.
      uint32_t pb[NT][NG][2];
      float t[NT][NG][2];
      auto weights = [&](auto anew) {
        bool over = false;
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float f = __fmul_rn(qs[n][i & 1], ks[b]), top = m[n][i & 1];
              if constexpr (decltype(anew)::value)  // (all of them -inf: P is 0)
                y[i] = __fadd_rn(__fsub_rn(__fmul_rn(s[b][n][i], f), top == -INFINITY ? 0.f : top), ve[b]);
              else
                y[i] = fmaf(s[b][n][i], f, ve[b] - top);
            }
            if (edge) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (tok_g + (i >> 1) * 8 >= valid[b]) y[i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = fast_exp2(y[i]);
            t[b][n][0] = y[0] + y[2];
            t[b][n][1] = y[1] + y[3];
            over |= fmaxf(t[b][n][0], t[b][n][1]) > 16384.f;
            pb[b][n][0] = pack_h2(y[0], y[1]);
            pb[b][n][1] = pack_h2(y[2], y[3]);
          }
        return over;
      };
      // (fresh: some maximum is -inf still)
      if (fresh || __any_sync(0xffffffffu, weights(std::false_type()))) {
        bool none = false;
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = m[n][c];
#pragma unroll
            for (int b = 0; b < NT; ++b) {
              const float f = __fmul_rn(qs[n][c], ks[b]);
              if (tok_g < valid[b]) mx = fmaxf(mx, __fmul_rn(s[b][n][c], f));
              if (tok_g + 8 < valid[b]) mx = fmaxf(mx, __fmul_rn(s[b][n][c + 2], f));
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float al = m[n][c] == mx ? 1.f : fast_exp2(m[n][c] - mx);
            m[n][c] = mx;
            none |= mx == -INFINITY;
            l[n][c] *= al;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              o[n][i][c] *= al;
              o[n][i][c + 2] *= al;
            }
          }
        fresh = __any_sync(0xffffffffu, none);
        weights(std::true_type());
      }
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        const float vu = fast_exp2(-ve[b]);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          l[n][0] = fmaf(t[b][n][0], vu, l[n][0]);
          l[n][1] = fmaf(t[b][n][1], vu, l[n][1]);
          pb[b][n][0] = movmatrix(pb[b][n][0]);
          pb[b][n][1] = movmatrix(pb[b][n][1]);
        }
      }
      // O^T += V^T P^T; rows past the last token may hold any bits
      if (edge) {
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (token_of<D>(2 * t4 + (i & 1)) + (i >> 1) * 8 >= valid[b])
#pragma unroll
              for (int w = 0; w < WR; ++w) v[b][i * WR + w] = 0u;
      }
      auto values = [&](auto scaled) {
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
          for (int w = 0; w < WR; ++w)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t sel = half ? 0x7362 : 0x5140;  // bytes (A0 B0 A1 B1) or (A2 B2 A3 B3)
              uint32_t a0, a1, a2, a3;
              e4m3x4_to_f16(__byte_perm(v[b][w], v[b][WR + w], sel), a0, a1);
              e4m3x4_to_f16(__byte_perm(v[b][2 * WR + w], v[b][3 * WR + w], sel), a2, a3);
              if constexpr (decltype(scaled)::value) {
                const __half2 f = __float2half2_rn(rest[b]);
                a0 = mul_h2(a0, f), a1 = mul_h2(a1, f), a2 = mul_h2(a2, f), a3 = mul_h2(a3, f);
              }
#pragma unroll
              for (int n = 0; n < NG; ++n) mma_f16(o[n][2 * w + half], a0, a1, a2, a3, pb[b][n][0], pb[b][n][1]);
            }
      };
      if (odd)
        values(std::true_type());
      else
        values(std::false_type());
      j += NT;
    };
    for (int tile = r0; tile < r1;) {
      if (tile == u.end) {
        end_unit();
        u = unit_at(tile);
        load_q();
        begin_unit();
      }
      const int before = j;
      // two tiles at once where the unit, the range and the 32 places have them: half the bookkeeping, twice the
      // independent work (D = 128 has that in one)
      if (D == 64 && min(u.end, r1) - tile >= 2 && j < 31) {
        attend(tile, std::integral_constant<int, D == 64 ? 2 : 1>());
        tile += 2;
      } else {
        attend(tile, std::integral_constant<int, 1>());
        ++tile;
      }
      if (j == 32) {
        j = 0;
        grp = grp_n;
        sc = sc_n;
        bad = __ballot_sync(0xffffffffu, missing);
        missing = false;
        grp_n = 0;
        if (tile + 32 + lane < r1) grp_n = find_tile(tile + 32 + lane, missing);
      } else if (before < 16 && j >= 16) {
        sc_n = scales(scales_raw(grp_n));
      }
    }
    if (late) atomicOr(a.err, MVB_DEV_TIMEOUT);
    __syncwarp();  // the ring has been read, and no copy is on its way: the last piece may lie in it
    end_unit();
  }
  __syncthreads();

  // ---- units cut inside this CTA: candidate w < NW began in warp w (pieces: its
  // slot 1, then slot 0 of the warps after it that hold the unit), candidate NW
  // began in an earlier CTA (pieces: slot 0 from warp 0 on) ----
  int* list = reinterpret_cast<int*>(pre);  // (the prefix is not needed any more) candidates, their numbers of pieces
  __shared__ int count;
  if (warp == 0) {
    const int4 id = lane < NW ? ids[lane * 2 + 1] : lane == NW ? ids[0] : make_int4(-1, 0, 0, 0);
    const int first = lane < NW ? lane + 1 : 0;  // slot 0 pieces from here on
    int n = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) n += w >= first && ids[w * 2].x == id.x;
    const uint32_t live = __ballot_sync(0xffffffffu, id.x >= 0);
    if (id.x >= 0) {
      const int at = __popc(live & ((1u << lane) - 1));
      list[2 * at] = lane;
      list[2 * at + 1] = n;
    }
    if (lane == 0) count = __popc(live);
    if (lane < 2) a.desc[blockIdx.x * 2 + lane] = make_int4(-1, 0, 0, 0);
  }
  __syncthreads();
  // D / 4 threads per head row, four columns each; pieces in warp order
  constexpr int TPR = D / 4, STEP = NW * 32 / TPR;
  for (int row = tid / TPR; row < count * HR; row += STEP) {
    const int at = row / HR, h = row - at * HR, d = (tid % TPR) * 4;
    const int cand = list[2 * at], n0 = list[2 * at + 1];
    const bool own = cand < NW;  // it has a slot 1
    const int4 id = own ? ids[cand * 2 + 1] : ids[0];
    const int kvh = id.z / a.head_groups, hg = id.z - kvh * a.head_groups;
    const int hb = kvh * a.G + hg * HR, n_h = min(HR, a.G - hg * HR);
    if (h >= n_h) continue;
    const float* p1 = part_of(own ? cand : 0, own ? 1 : 0);
    const float* p0 = part_of(own ? cand + 1 : 0, 0);
    constexpr int STRIDE = Sm::PIECE / 4;
    float M = own ? p1[HR * D + 2 * h] : -INFINITY;
#pragma unroll 4
    for (int w = 0; w < n0; ++w) M = fmaxf(M, p0[w * STRIDE + HR * D + 2 * h]);
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float* p) {
      const float2 ml = *reinterpret_cast<const float2*>(p + HR * D + 2 * h);
      const float4 o = *reinterpret_cast<const float4*>(p + h * D + d);
      const float w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
      L = fmaf(w, ml.y, L);
      acc = make_float4(fmaf(w, o.x, acc.x), fmaf(w, o.y, acc.y), fmaf(w, o.z, acc.z), fmaf(w, o.w, acc.w));
    };
    if (own) add(p1);
#pragma unroll 4
    for (int w = 0; w < n0; ++w) add(p0 + w * STRIDE);
    if (own && id.w != 0) {
      const float f = L == 0.f ? 0.f : 1.f / L;
      uint2 w;
      T* e = reinterpret_cast<T*>(&w);
      e[0] = from_f32<T>(acc.x * f), e[1] = from_f32<T>(acc.y * f);
      e[2] = from_f32<T>(acc.z * f), e[3] = from_f32<T>(acc.w * f);
      *reinterpret_cast<uint2*>(out + (int64_t)id.y * a.o_s0 + (int64_t)(hb + h) * a.o_s1 + d) = w;
    } else {
      const int slot = own ? 1 : 0;
      float* p = a.part + ((int64_t)blockIdx.x * 2 + slot) * 16 * (D + 2);
      *reinterpret_cast<float4*>(p + h * D + d) = acc;
      if (d == 0) {
        *reinterpret_cast<float2*>(p + HR * D + 2 * h) = make_float2(M, L);
        if (h == 0) a.desc[blockIdx.x * 2 + slot] = make_int4(id.x, id.y, hb, n_h);
      }
    }
  }
}

// Joins the partial states of units cut between CTAs: CTA c takes the unit that
// begins in stream CTA c and runs on; one head row per warp and step, pieces in
// CTA order, 32 at a time.
template <typename T, int D, int HR>
__global__ void __launch_bounds__(256) fp8_decode_merge_kernel(const Fp8DecodeArgs a, int ctas) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 id = __ldcg(a.desc + c * 2 + 1);
  if (id.x < 0) return;
  int n = 1;  // pieces: CTA c's slot 1, then slot 0 of the CTAs after it
  for (int i = c + 1; i < ctas; i += 32) {
    const bool same = i + lane < ctas && __ldcg(a.desc + (i + lane) * 2).x == id.x;
    const uint32_t other = ~__ballot_sync(0xffffffffu, same);
    const int run = other ? __ffs(other) - 1 : 32;
    n += run;
    if (run < 32) break;
  }
  auto piece = [&](int i) { return a.part + ((int64_t)(c + i) * 2 + (i == 0 ? 1 : 0)) * 16 * (D + 2); };
  for (int h = warp; h < id.w; h += 8) {
    float M = -INFINITY;
    for (int i = lane; i < n; i += 32) M = fmaxf(M, __ldcg(piece(i) + HR * D + 2 * h));
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
    float L = 0.f, acc[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
    for (int i0 = 0; i0 < n; i0 += 32) {
      float w = 0.f, x = 0.f;
      if (i0 + lane < n) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(piece(i0 + lane) + HR * D + 2 * h));
        w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
        x = w * ml.y;
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
      L += x;
#pragma unroll 4
      for (int i = i0; i < min(n, i0 + 32); ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i - i0);
        const float* p = piece(i) + h * D;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(wi, __ldcg(p + lane + 32 * e), acc[e]);
      }
    }
    const float f = L == 0.f ? 0.f : 1.f / L;
    T* p = static_cast<T*>(a.out) + (int64_t)id.y * a.o_s0 + (int64_t)(id.z + h) * a.o_s1;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) p[lane + 32 * e] = from_f32<T>(acc[e] * f);
  }
}

// CTAs of the stream kernel: one per SM, fewer where the tables bound the work; or one per unit.
int decode_grid(int num_seqs, int units_per_seq, int max_blocks, int block_size, int nw, int* whole) {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t units = (int64_t)num_seqs * units_per_seq, unit_tiles = (int64_t)max_blocks * block_size / kFp8Tile;
  const int64_t mine = (unit_tiles + nw - 1) / nw, share = std::max<int64_t>(kFp8MinTiles, units * unit_tiles / (sms * nw));
  *whole = units <= sms && mine <= kFp8WholeTiles && mine - share <= kFp8WholeMore;
  if (*whole) return (int)std::max<int64_t>(units, 1);
  const int64_t tiles = units * unit_tiles;
  const int64_t per = (int64_t)nw * kFp8MinTiles;
  const int64_t want = (tiles + per - 1) / per;
  return (int)(want < 1 ? 1 : want < sms ? want : sms);
}

struct Fp8DecodePlan {
  int head_groups, ng, nw, grid, whole;
  int64_t off_part, bytes;
};

int plan_decode(int num_seqs, int num_heads, int num_kv_heads, int head_dim, int block_size, int num_blocks,
                int max_blocks, int dtype, Fp8DecodePlan* pl) {
  if (dtype != MVB_DTYPE_F16 && dtype != MVB_DTYPE_BF16) return MVB_ERR_DTYPE;
  if (head_dim != 64 && head_dim != 128) return MVB_ERR_HEAD_DIM;
  if (block_size < kFp8MinBlock || block_size > kFp8MaxBlock || (block_size & (block_size - 1)) != 0)
    return MVB_ERR_BLOCK_SIZE;
  if (num_seqs < 0 || num_seqs > kFp8DecodeMaxSeqs || num_heads <= 0 || num_kv_heads <= 0 || num_blocks <= 0 ||
      max_blocks < 0)
    return MVB_ERR_INVALID_ARG;
  if (num_heads % num_kv_heads != 0) return MVB_ERR_HEADS;
  const int G = num_heads / num_kv_heads;
  pl->ng = G > 8 ? 2 : 1;
  pl->head_groups = (G + 8 * pl->ng - 1) / (8 * pl->ng);
  pl->nw = head_dim == 64 ? (pl->ng == 1 ? Fp8Geo<64, 1>::NW : Fp8Geo<64, 2>::NW)
                          : (pl->ng == 1 ? Fp8Geo<128, 1>::NW : Fp8Geo<128, 2>::NW);
  const int units = num_kv_heads * pl->head_groups;
  // tile and cache row numbers are 32-bit
  if ((int64_t)num_seqs * units * ((int64_t)max_blocks * block_size / kFp8Tile + 1) >= ((int64_t)1 << 31) ||
      (int64_t)num_blocks * num_kv_heads * block_size >= ((int64_t)1 << 31))
    return MVB_ERR_INVALID_ARG;
  pl->grid = decode_grid(num_seqs, units, max_blocks, block_size, pl->nw, &pl->whole);
  pl->off_part = ((int64_t)pl->grid * 32 + 255) / 256 * 256;
  pl->bytes = pl->off_part + (int64_t)pl->grid * 2 * 16 * (head_dim + 2) * 4;
  return MVB_OK;
}

// A cache of `bytes` bytes as rows of 128, a 16-token tile a box.
bool cache_map(const void* base, int64_t bytes, int head_dim, CUtensorMap* map) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {128, (cuuint64_t)(bytes / 128)};
  const cuuint64_t strides[1] = {128};
  const cuuint32_t box[2] = {128, (cuuint32_t)(kFp8Tile * head_dim / 128)};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, int NG>
int launch_decode(const Fp8DecodeArgs& a, int grid, cudaStream_t stream) {
  CUtensorMap tmk, tmv;
  const int64_t bytes = (((int64_t)a.num_blocks * a.num_kv_heads) << a.block_shift) * D;
  if (!cache_map(a.kc, bytes, D, &tmk) || !cache_map(a.vc, bytes, D, &tmv)) return MVB_ERR_TENSOR_MAP;
  auto kern = fp8_decode_kernel<T, D, NG>;
  const int smem = Fp8Smem<D, NG>::bytes(a.num_seqs);
  // the largest batch's size at once: the attribute is set on the first call only
  if (ensure_kernel_attrs(kern, Fp8Smem<D, NG>::bytes(kFp8DecodeMaxSeqs)) != cudaSuccess) return MVB_ERR_CUDA;
  if (launch_pdl(kern, dim3(grid), dim3(Fp8Geo<D, NG>::NW * 32), smem, stream, tmk, tmv, a) != cudaSuccess) return MVB_ERR_CUDA;
  if (grid == 1 || a.whole) return MVB_OK;  // no unit is cut between CTAs
  auto merge = fp8_decode_merge_kernel<T, D, 8 * NG>;
  if (ensure_kernel_attrs(merge, 0) != cudaSuccess) return MVB_ERR_CUDA;
  return launch_pdl(merge, dim3(grid), dim3(256), 0, stream, a, grid) == cudaSuccess ? MVB_OK : MVB_ERR_CUDA;
}

template <typename T>
int launch_decode_t(const Fp8DecodeArgs& a, int head_dim, const Fp8DecodePlan& pl, cudaStream_t stream) {
  if (head_dim == 64)
    return pl.ng == 1 ? launch_decode<T, 64, 1>(a, pl.grid, stream) : launch_decode<T, 64, 2>(a, pl.grid, stream);
  return pl.ng == 1 ? launch_decode<T, 128, 1>(a, pl.grid, stream) : launch_decode<T, 128, 2>(a, pl.grid, stream);
}

}  // namespace
}  // namespace mvb

using namespace mvb;

extern "C" int mvb_paged_decode_fp8_workspace(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
                                              int32_t head_dim, int32_t block_size, int32_t num_blocks,
                                              int32_t max_blocks_per_seq, int32_t dtype, int64_t* bytes_out) {
  Fp8DecodePlan pl;
  const int st = plan_decode(num_seqs, num_heads, num_kv_heads, head_dim, block_size, num_blocks, max_blocks_per_seq,
                             dtype, &pl);
  if (st == MVB_OK && bytes_out) *bytes_out = pl.bytes;
  return st;
}

extern "C" int mvb_paged_decode_fp8(const void* query, int64_t q_stride_seq, int64_t q_stride_head,
                                    const void* key_cache, const void* value_cache, const float* kv_scale,
                                    const int64_t* block_table, int64_t block_table_stride,
                                    int32_t max_blocks_per_seq, const int32_t* kv_len, void* out,
                                    int64_t out_stride_seq, int64_t out_stride_head, int32_t num_seqs,
                                    int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                    int32_t num_blocks, float scale, int32_t dtype, void* workspace,
                                    int64_t workspace_bytes, int32_t* error_flags, void* stream) {
  mvb::NvtxRange nvtx_range("mvb_paged_decode_fp8");
  Fp8DecodePlan pl;
  const int st = plan_decode(num_seqs, num_heads, num_kv_heads, head_dim, block_size, num_blocks, max_blocks_per_seq,
                             dtype, &pl);
  if (st != MVB_OK) return st;
  if (num_seqs == 0) return MVB_OK;
  if (!query || !key_cache || !value_cache || !kv_scale || !block_table || !kv_len || !out || !error_flags)
    return MVB_ERR_INVALID_ARG;
  if (max_blocks_per_seq > 0 && block_table_stride < max_blocks_per_seq) return MVB_ERR_INVALID_ARG;
  auto al = [](const void* p, int64_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  if (!al(query, 16) || q_stride_seq % 8 || q_stride_head % 8 || !al(out, 16) || out_stride_seq % 8 ||
      out_stride_head % 8 || !al(key_cache, 16) || !al(value_cache, 16) || !al(kv_scale, 8))
    return MVB_ERR_ALIGNMENT;
  if (workspace == nullptr || workspace_bytes < pl.bytes || !al(workspace, 256)) return MVB_ERR_WORKSPACE;
  Fp8DecodeArgs a;
  a.q = query;
  a.q_s0 = q_stride_seq;
  a.q_s1 = q_stride_head;
  a.kc = static_cast<const uint8_t*>(key_cache);
  a.vc = static_cast<const uint8_t*>(value_cache);
  a.scale = reinterpret_cast<const float2*>(kv_scale);
  a.bt = block_table;
  a.bt_s0 = block_table_stride;
  a.max_blocks = max_blocks_per_seq;
  a.kv_len = kv_len;
  a.out = out;
  a.o_s0 = out_stride_seq;
  a.o_s1 = out_stride_head;
  a.num_seqs = num_seqs;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.G = num_heads / num_kv_heads;
  a.head_groups = pl.head_groups;
  a.whole = pl.whole;
  a.block_shift = 31 - __builtin_clz(block_size);
  a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.desc = static_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + pl.off_part);
  a.err = error_flags;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MVB_DTYPE_BF16 ? launch_decode_t<__nv_bfloat16>(a, head_dim, pl, s)
                                 : launch_decode_t<__half>(a, head_dim, pl, s);
}
