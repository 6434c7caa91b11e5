// Generic paged decode attention on CUDA cores: any head_dim <= 512, any storage
// type, any GQA ratio, explicit or sliding window. One block per
// (q head, split, sequence); warps stride over rows, lanes over dims; online
// softmax in the log2 domain; the block that arrives last for a q head merges the
// split partials. It is the path for f32 pages and for shapes the tensor-core
// kernel does not take, and it cross-checks that kernel in the tests. Computes
// what attention_decode_naive/flash compute (src/decode_resident/kernels.rs:11-366).
#include "kernels.h"

namespace sgk {

constexpr int GEN_THREADS = 128;
constexpr int GEN_WARPS = GEN_THREADS / 32;
constexpr int GEN_MAXJ = 16;  // head_dim <= 32 * 16

// U4, SINKS: instances for u4 pages and for sinks beside a window, so that neither costs the others anything.
template <bool U4, bool SINKS>
__global__ void __launch_bounds__(GEN_THREADS) attention_generic_kernel(AttnArgs a) {
  extern __shared__ float smem[];
  const int hd = a.pool.head_dim;
  float* q_s = smem;                       // [hd]
  float* o_s = smem + hd;                  // [GEN_WARPS][hd]
  float* ml_s = o_s + GEN_WARPS * hd;      // [GEN_WARPS][2]
  __shared__ int is_last_s;

  const int qh = blockIdx.x, split = blockIdx.y, seq = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gqa = a.q_heads / a.pool.kv_heads;
  const int kvh = qh / gqa;
  const int slot = a.slots ? a.slots[seq] : a.slot0;
  const int64_t len = a.pool.lens[int64_t(slot) * a.pool.layers + a.layer];
  int64_t ws = a.sliding_window > 0 ? (len > a.sliding_window ? len - a.sliding_window : 0) : a.window_start;
  if (ws > len) ws = len;
  // visible rows: `sinks` at the head, then [ws, len); i counts them, row i + (i < sinks ? 0 : gap)
  const int64_t sinks = !SINKS ? 0 : a.sink_rows < ws ? a.sink_rows : ws;
  const int64_t gap = ws - sinks;
  const int64_t n = len - gap;
  const int64_t i0 = (n * split) / a.splits;
  const int64_t i1 = (n * (split + 1)) / a.splits;
  const int32_t* table = a.pool.tables + int64_t(slot) * a.pool.table_stride;

  const float* q = a.q + (int64_t(seq) * a.q_heads + qh) * hd;
  for (int c = tid; c < hd; c += GEN_THREADS) q_s[c] = q[c] * a.scale_log2e;
  __syncthreads();

  float m = -1.0e30f, l = 0.0f;
  float acc[GEN_MAXJ];
#pragma unroll
  for (int j = 0; j < GEN_MAXJ; ++j) acc[j] = 0.0f;

  if constexpr (U4 || SINKS) {
    // ROWS rows at a time: their table entries, keys and values are asked for together, and the reductions of their
    // products overlap (u4, one row after the other and four at a time: 43 sequences of 96 rows, 32/4 heads of 64, 58.0 and
    // 55.9 us; 10 of 4000 to 8000 rows, 8/1 heads of 96, 230 and 224)
    constexpr int ROWS = 4;
    for (int64_t i = i0 + warp * ROWS; i < i1; i += GEN_WARPS * ROWS) {
      const uint8_t* ktile[ROWS];
      int rin[ROWS];
      bool on[ROWS];
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const int64_t v = i + u < i1 ? i + u : i;
        const int64_t r = SINKS && v < sinks ? v : v + gap;
        const int32_t page = table[r / PAGE_TOKENS];
        on[u] = i + u < i1 && page >= 0 && page < a.num_pages;
        if (i + u < i1 && !on[u] && lane == 0) atomicExch(a.status, DEV_ERR_BAD_PAGE);
        rin[u] = static_cast<int>(r % PAGE_TOKENS);
        ktile[u] = a.pool.base + tile_offset(a.pool, page >= 0 && page < a.num_pages ? page : 0, a.layer, kvh, 0);
      }
      float dot[ROWS];
#pragma unroll
      for (int u = 0; u < ROWS; ++u) dot[u] = 0.0f;
#pragma unroll
      for (int j = 0; j < GEN_MAXJ; ++j) {
        const int d = lane + 32 * j;
        if (32 * j >= hd) break;   // uniform
        if (d < hd) {
#pragma unroll
          for (int u = 0; u < ROWS; ++u)
            dot[u] += q_s[d] * (U4 ? load_u4_elem(ktile[u], hd, 0, rin[u], d) : load_tile_elem(ktile[u], a.pool.dtype, hd, 0, rin[u], d));
        }
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1)
#pragma unroll
        for (int u = 0; u < ROWS; ++u) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], off);
      float m_new = m;
#pragma unroll
      for (int u = 0; u < ROWS; ++u)
        if (on[u]) m_new = fmaxf(m_new, dot[u]);
      const float alpha = exp2f(m - m_new);
      float p[ROWS];
      l *= alpha;
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        p[u] = on[u] ? exp2f(dot[u] - m_new) : 0.0f;
        l += p[u];
      }
#pragma unroll
      for (int j = 0; j < GEN_MAXJ; ++j) {
        const int d = lane + 32 * j;
        if (32 * j >= hd) break;   // uniform
        if (d < hd) {
          float sum = acc[j] * alpha;
#pragma unroll
          for (int u = 0; u < ROWS; ++u) {
            const uint8_t* vtile = ktile[u] + a.pool.tile_bytes;
            const float x = U4 ? load_u4_elem(vtile, hd, 1, rin[u], d) : load_tile_elem(vtile, a.pool.dtype, hd, 1, rin[u], d);
            sum += on[u] ? p[u] * x : 0.0f;
          }
          acc[j] = sum;
        }
      }
      m = m_new;
    }
  } else {
  for (int64_t i = i0 + warp; i < i1; i += GEN_WARPS) {
    const int64_t r = i + gap;
    int32_t page = table[r / PAGE_TOKENS];
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0) atomicExch(a.status, DEV_ERR_BAD_PAGE);
      continue;
    }
    const int rin = static_cast<int>(r % PAGE_TOKENS);
    const uint8_t* ktile = a.pool.base + tile_offset(a.pool, page, a.layer, kvh, 0);
    const uint8_t* vtile = ktile + a.pool.tile_bytes;
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < GEN_MAXJ; ++j) {
      int d = lane + 32 * j;
      if (d < hd) dot += q_s[d] * load_tile_elem(ktile, a.pool.dtype, hd, 0, rin, d);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    float m_new = fmaxf(m, dot);
    float alpha = exp2f(m - m_new);
    float p = exp2f(dot - m_new);
    l = l * alpha + p;
#pragma unroll
    for (int j = 0; j < GEN_MAXJ; ++j) {
      int d = lane + 32 * j;
      if (d < hd) acc[j] = acc[j] * alpha + p * load_tile_elem(vtile, a.pool.dtype, hd, 1, rin, d);
    }
    m = m_new;
  }
  }

  // merge the warps of this block
#pragma unroll
  for (int j = 0; j < GEN_MAXJ; ++j) {
    int d = lane + 32 * j;
    if (d < hd) o_s[warp * hd + d] = acc[j];
  }
  if (lane == 0) {
    ml_s[2 * warp] = m;
    ml_s[2 * warp + 1] = l;
  }
  __syncthreads();
  float mb = -1.0e30f;
#pragma unroll
  for (int w = 0; w < GEN_WARPS; ++w) mb = fmaxf(mb, ml_s[2 * w]);
  float lb = 0.0f;
  float wgt[GEN_WARPS];
#pragma unroll
  for (int w = 0; w < GEN_WARPS; ++w) {
    wgt[w] = exp2f(ml_s[2 * w] - mb);
    lb += ml_s[2 * w + 1] * wgt[w];
  }
  const int64_t qh_global = int64_t(seq) * a.q_heads + qh;
  float* out_row = a.out + qh_global * hd;
  if (a.splits == 1) {
    float inv = 1.0f / lb;
    for (int d = tid; d < hd; d += GEN_THREADS) {
      float o = 0.0f;
#pragma unroll
      for (int w = 0; w < GEN_WARPS; ++w) o += o_s[w * hd + d] * wgt[w];
      out_row[d] = o * inv;
    }
    return;
  }
  float* po = a.part.o + (qh_global * a.splits + split) * hd;
  for (int d = tid; d < hd; d += GEN_THREADS) {
    float o = 0.0f;
#pragma unroll
    for (int w = 0; w < GEN_WARPS; ++w) o += o_s[w * hd + d] * wgt[w];
    po[d] = o;
  }
  if (tid == 0) {
    float* pml = a.part.ml + (qh_global * a.splits + split) * 2;
    pml[0] = mb;
    pml[1] = lb;
  }
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    int old = atomicAdd(a.head_counters + qh_global, 1);
    is_last_s = (old == a.splits - 1);
  }
  __syncthreads();
  if (is_last_s) {
    __threadfence();
    merge_partials(a.part, qh_global, a.splits, hd, out_row, tid, GEN_THREADS);
    if (tid == 0) a.head_counters[qh_global] = 0;
  }
}

cudaError_t launch_attention_generic(const AttnArgs& a, int n_seq, cudaStream_t stream) {
  dim3 grid(a.q_heads, a.splits, n_seq);
  size_t smem = (size_t(a.pool.head_dim) * (1 + GEN_WARPS) + 2 * GEN_WARPS) * sizeof(float);
  const bool u4 = a.pool.dtype == KV_U4G32, sinks = a.sink_rows > 0;
  if (u4 && sinks) attention_generic_kernel<true, true><<<grid, GEN_THREADS, smem, stream>>>(a);
  else if (u4) attention_generic_kernel<true, false><<<grid, GEN_THREADS, smem, stream>>>(a);
  else if (sinks) attention_generic_kernel<false, true><<<grid, GEN_THREADS, smem, stream>>>(a);
  else attention_generic_kernel<false, false><<<grid, GEN_THREADS, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace sgk
