// mvb_paged_prefill_fp8: causal attention of a batch of prefill chunks over an
// 8-bit paged cache (codes with a scale per (block, KV head)); the chunk's own
// tokens are in the cache before the call.  Query token t of a chunk with c
// cached tokens attends positions [0, c + t].
//
// The rows of one KV head are (token, head of its group) pairs, token-major, so
// that the query heads that share keys share a tile.  One warp holds 16 rows as
// the columns of S^T = K Q^T (the math of the decode kernel, fp8_decode.cu) and
// walks the 16-token tiles up to its last row's limit.
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
constexpr int kRows = 128;  // (token, head) rows of one CTA
constexpr int kWarps = 8;

__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32, 1) fp8_prefill_kernel(const Fp8PrefillArgs a) {
  constexpr int NG = 2, MT = D / 16, KS = D / 16, KW = D / 64, NT = kWarps * 32;
  extern __shared__ int pre[];  // [n + 1] row-tile prefix, then [n + 1] token prefix
  int* qpre = pre + a.n + 1;
  __shared__ int s_tot[2][kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  grid_dependency_wait();
  grid_launch_dependents();
  {
    const int per = (a.n + NT - 1) / NT;
    const int i0 = min(a.n, tid * per), i1 = min(a.n, i0 + per);
    int mt = 0, mq = 0;
    for (int i = i0; i < i1; ++i) {
      const int ql = (int)min((int64_t)a.total_q + 1, max((int64_t)0, __ldg(a.qlen + i)));
      pre[i] = (int)(((int64_t)ql * a.G + kRows - 1) / kRows);
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
        iq += vq;
      }
    }
    if (lane == 31) {
      s_tot[0][warp] = it;
      s_tot[1][warp] = iq;
    }
    __syncthreads();
    int rt = it - mt, rq = iq - mq, Tt = 0, Tq = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) {
        rt += s_tot[0][w];
        rq += s_tot[1][w];
      }
      Tt += s_tot[0][w];
      Tq += s_tot[1][w];
    }
    for (int i = i0; i < i1; ++i) {
      const int t = pre[i], q = qpre[i];
      pre[i] = rt;
      qpre[i] = rq;
      rt += t;
      rq += q;
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
  const int x = blockIdx.x;
  if (x >= pre[a.n]) return;
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
  const int row0 = (x - pre[lo]) * kRows + warp * 16;  // the warp's first row in the chunk
  const int64_t srow = __ldg(a.seq_rows + lo), cached = __ldg(a.cached + lo);
  T* const out = static_cast<T*>(a.out);
  const bool bad = cached < 0 || srow < 0 || srow >= a.bt_rows ||
                   (cached + ql + (1 << a.block_shift) - 1) >> a.block_shift > a.max_blocks;
  if (row0 >= rows) return;
  if (bad) {
    if (lane == 0) atomicOr(a.err, MVB_DEV_TABLE_SHORT);
    for (int e = lane; e < min(16, rows - row0) * D; e += 32) {
      const int r = row0 + e / D;
      out[(int64_t)(q0 + r / a.G) * a.o_s0 + (int64_t)(h0 + r % a.G) * a.o_s1 + e % D] = from_f32<T>(0.f);
    }
    return;
  }
  uint32_t qf[NG][KS][2];
  float qs[NG][2], o[NG][MT][4], m[NG][2], l[NG][2];
  int lim[NG][2];  // positions this lane's columns (rows row0 + 8n + 2t, + 1) attend
  int last = 0;    // the warp's largest
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    const int r = row0 + 8 * n + g;
    const bool live = r < rows;
    const T* qp = static_cast<const T*>(a.q) + (int64_t)(q0 + r / a.G) * a.q_s0 + (int64_t)(h0 + r % a.G) * a.q_s1;
    float xv[KW][16], amax = 0.f;
#pragma unroll
    for (int c = 0; c < KW; ++c) {
      uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      if (live) {
        raw[0] = __ldg(reinterpret_cast<const uint4*>(qp + 64 * c + 16 * t4));
        raw[1] = __ldg(reinterpret_cast<const uint4*>(qp + 64 * c + 16 * t4) + 1);
      }
      const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        xv[c][i] = to_f32<T>(e[i]);
        const float y = fabsf(xv[c][i]);
        amax = fmaxf(amax, y < INFINITY ? y : 0.f);
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int e = min(max((int)(__float_as_uint(amax) >> 23), 2), 252);
    const float down = __uint_as_float((uint32_t)(254 - e) << 23), up = __uint_as_float((uint32_t)e << 23);
#pragma unroll
    for (int c = 0; c < KW; ++c)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        qf[n][4 * c + k][0] = pack_h2(xv[c][4 * k] * down, xv[c][4 * k + 1] * down);
        qf[n][4 * c + k][1] = pack_h2(xv[c][4 * k + 2] * down, xv[c][4 * k + 3] * down);
      }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      qs[n][c] = a.scale_log2 * __shfl_sync(0xffffffffu, up, (2 * t4 + c) * 4);
      const int rc = row0 + 8 * n + 2 * t4 + c;
      lim[n][c] = rc < rows ? (int)cached + rc / a.G + 1 : 0;
      m[n][c] = -INFINITY;
      l[n][c] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
  }
  last = (int)cached + (min(row0 + 16, rows) - 1) / a.G + 1;
  const int64_t* bt = a.bt + srow * a.bt_s0;
  for (int t0 = 0; t0 < last; t0 += 16) {
    const int64_t b = __ldg(bt + (t0 >> a.block_shift));
    if (b < 0 || b >= a.num_blocks) {
      if (lane == 0) atomicOr(a.err, MVB_DEV_BLOCK_ID);
      continue;
    }
    const int64_t bh = b * a.num_kv_heads + kvh;
    const float2 sc = __ldg(a.scale + bh);
    const int64_t off = ((bh << a.block_shift) + (t0 & ((1 << a.block_shift) - 1))) * D;
    const uint8_t* kp = a.kc + off + 16 * t4;
    const uint8_t* vp = a.vc + off + 2 * t4 * D + (D / 8) * g;
    float s[NG][4];
#pragma unroll
    for (int n = 0; n < NG; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int c = 0; c < KW; ++c) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(kp + g * D + 64 * c));
      const uint4 y = __ldg(reinterpret_cast<const uint4*>(kp + (g + 8) * D + 64 * c));
      const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a0, a1, a2, a3;
        e4m3x4_to_f16(xw[k], a0, a2);
        e4m3x4_to_f16(yw[k], a1, a3);
#pragma unroll
        for (int n = 0; n < NG; ++n) mma_f16(s[n], a0, a1, a2, a3, qf[n][4 * c + k][0], qf[n][4 * c + k][1]);
      }
    }
    uint32_t pb[NG][2];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float f = qs[n][c] * sc.x;
        const float x0 = t0 + g < lim[n][c] ? s[n][c] * f : -INFINITY;
        const float x1 = t0 + g + 8 < lim[n][c] ? s[n][c + 2] * f : -INFINITY;
        float mx = fmaxf(x0, x1);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        mx = fmaxf(mx, m[n][c]);
        const float al = m[n][c] == mx ? 1.f : fast_exp2(m[n][c] - mx);
        m[n][c] = mx;
        s[n][c] = x0 == -INFINITY ? 0.f : fast_exp2(x0 - mx);
        s[n][c + 2] = x1 == -INFINITY ? 0.f : fast_exp2(x1 - mx);
        l[n][c] = l[n][c] * al + s[n][c] + s[n][c + 2];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          o[n][i][c] *= al;
          o[n][i][c + 2] *= al;
        }
      }
      pb[n][0] = movmatrix(pack_h2(s[n][0], s[n][1]));
      pb[n][1] = movmatrix(pack_h2(s[n][2], s[n][3]));
    }
    // rows past the warp's last limit may hold any bits
    constexpr int WR = D / 32;
    uint32_t v[4][WR];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = (i & 1) + (i >> 1) * 8;
      const bool ok = t0 + 2 * t4 + r < last;
#pragma unroll
      for (int w = 0; w < WR; ++w)
        v[i][w] = ok ? __ldg(reinterpret_cast<const uint32_t*>(vp + r * D) + w) : 0u;
    }
#pragma unroll
    for (int w = 0; w < WR; ++w)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t sel = half ? 0x7362 : 0x5140;
        uint32_t a0, a1, a2, a3;
        e4m3x4_to_f16(__byte_perm(v[0][w], v[1][w], sel), a0, a1);
        e4m3x4_to_f16(__byte_perm(v[2][w], v[3][w], sel), a2, a3);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          float y[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16(y, a0, a1, a2, a3, pb[n][0], pb[n][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][2 * w + half][e] = fmaf(y[e], sc.y, o[n][2 * w + half][e]);
        }
      }
  }
#pragma unroll
  for (int n = 0; n < NG; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float s = l[n][c];
      s += __shfl_xor_sync(0xffffffffu, s, 4);
      s += __shfl_xor_sync(0xffffffffu, s, 8);
      s += __shfl_xor_sync(0xffffffffu, s, 16);
      const int r = row0 + 8 * n + 2 * t4 + c;
      if (r >= rows) continue;
      const float inv = s == 0.f ? 0.f : 1.f / s;
      T* p = out + (int64_t)(q0 + r / a.G) * a.o_s0 + (int64_t)(h0 + r % a.G) * a.o_s1 + (D / 8) * g;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        p[2 * i] = from_f32<T>(o[n][i][c] * inv);
        p[2 * i + 1] = from_f32<T>(o[n][i][c + 2] * inv);
      }
    }
}

template <typename T, int D>
int launch_prefill_fp8(const Fp8PrefillArgs& a, cudaStream_t stream) {
  auto kern = fp8_prefill_kernel<T, D>;
  const int smem = 2 * (a.n + 1) * 4;
  if (ensure_kernel_attrs(kern, smem) != cudaSuccess) return MVB_ERR_CUDA;
  const int64_t tiles = ((int64_t)a.total_q * a.G + kRows - 1) / kRows + a.n;
  return launch_pdl(kern, dim3((unsigned)tiles, a.num_kv_heads), dim3(kWarps * 32), smem, stream, a) == cudaSuccess
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
