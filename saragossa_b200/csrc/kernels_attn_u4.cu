// Paged split-K flash-decoding over u4 group-32 pages (head_dim 64 / 128 / 256, GQA group <= 8), with the
// per-token append (quantisation included) fused in and with attention sinks beside the window.
//
// One block per (split, kv head, sequence); every warp of a block fetches pages of its own (one bulk async copy per page
// into its part of a shared-memory ring) and the partial results meet in the merges that the other paged kernels use.
// A page is worth 5/16 of its bf16 bytes and nearly the same products, so here the warps' instructions count:
//
//   codes    a byte holds two codes, n0 + 16 n1 (dims p and p + 16); a word becomes four registers of fp16 numbers, the
//            bytes u = n0 + 16 n1 and the low codes n0, with six instructions (U4Word). n0 x + n1 y = n0 (x - y / 16) + u (y / 16).
//   scores   the query is prepared once per launch as x - y / 16 and y / 16, fp16 hi + lo parts (22 bits; scaled by a power
//            of two per head, so any size of query keeps them). Products per group of 32 dims, then in f32
//              z[row][h] = sum_g step_k[row][g] (sum_d codes q) + sum_g bias_k[row][g] qsum[h][g] + e[row],
//            the bias sum as one bf16 product with qsum in three bf16 parts (24 bits).
//   softmax  a V row's steps are stored as f * 2^e with fp16 f (layout.h); 2^e joins the score, so the weight
//            p'' = exp2(z - M) is bounded whatever the row's range, and w = p'' f needs no scaling. p = p'' 2^-e
//            feeds the sum of the weights and the bias part of V. M is a reference, not the maximum: it moves only
//            when a z exceeds it by more than 14.9 (then to 9 or 10 below the largest z), so a page costs one vote
//            instead of the shuffles of a maximum, and p'' stays inside fp16.
//   classes  That holds while the 2^e of the rows lie within a factor of 16. One row of a wide range would raise M for all: the
//            others' weights would leave fp16 at its lower end, in the groups too where that row says nothing. So M belongs
//            to a class of rows: the vote also asks for rows with a 2^e below the class, and an iteration that meets rows of
//            another class goes through its pages once per class, M moving with the class by the exact power of two. A
//            row's weights are then off by 2^-28 of 2^e and of the largest weight at most: the codes of a group whose
//            step is 2^-k of the widest of its row by 2^(k-28) of their share (k <= 16), everything else by less than the scores.
//   outputs  O[d][h] = sum_row code w with w as fp16 hi + lo (22 bits; one part of 11 bits would leave 1e-4 of the result).
//
// Rows of odd position are stored negated (u4_quant.cuh): without it O would be a sum of codes that
// all count up from a minimum, hundreds of times larger than the result under flat attention, and f32
// would lose those digits.
//
// B200, one call after another on one stream, f32 queries, 32 query heads over 4 KV heads of 128: 8 sequences of 32768 rows
// 51.5 us = 3.3 TB/s of page bytes (50 % of the copy rate; DRAM reads 1.013 of the page bytes), one sequence 16.7 us; 24 uneven
// sequences of 200 to 20000 rows, 32 over 8 heads, 41.0 us = 3.4 TB/s; 64 windows of 2000 rows, 16 over 2 heads of 256, 32.2 us =
// 2.6 TB/s. No unit is full (8 x 32768: tensor pipe 33 %, ALU 27 %, DRAM 50 %; 0.44 instructions issued per scheduler and cycle,
// 345 per page and KV head): with two warps per scheduler the bound is latency, first the fixed latencies between
// dependent instructions (1.25 warps waiting per issue), then, below about 10 MB, start and merge.
// With V rows 10^6 times the others': one of them, or the first four rows a hundredth of the others, 54 us; one in 64, 91 us;
// every second one, 107 us.
//
// The reference's KV has no 4-bit form; this kernel computes cached_attention_one
// (src/decoder/attention_ops.rs:889-974) over the rows' values code * scale + bias.
#include "mma_common.cuh"
#include "u4_quant.cuh"

namespace sgk {

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same onto nothing: c = a b
__device__ __forceinline__ void mma_f16_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// 2^x; results below 2^-126 are zero
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_bf16_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ uint32_t pack_bf16(float x0, float x1) {  // x0 in the low half
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x1), "f"(x0));
  return r;
}
__device__ __forceinline__ float bf16_lo_f32(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float bf16_hi_f32(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_f16(float x0, float x1) {
  __half2 v = __floats2half2_rn(x0, x1);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
__device__ __forceinline__ uint32_t hmul2_u32(uint32_t a, uint32_t b) {
  __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hsub2_u32(uint32_t a, uint32_t b) {
  __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hfma2_u32(uint32_t a, uint32_t b, uint32_t c) {   // a b + c
  __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), *reinterpret_cast<__half2*>(&c));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hfms2_u32(uint32_t a, uint32_t b, uint32_t c) {   // a b - c
  __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), __hneg2(*reinterpret_cast<__half2*>(&c)));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {   // (a & b) | c as one instruction
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// A word's eight codes as four A registers: bytes 0, 2 and bytes 1, 3, as whole bytes u = 16 n1 + n0 and as low codes n0.
// u goes to the matrix unit as the fp16 subnormal u * 2^-24: one mask or permute. n0 must be a normal number,
// (1024 + n0) - 1024: the unit aligns its products by their exponent fields, and a subnormal's field lies up to ten
// bits above its value, digits that the accumulator loses. u is largest in the field and its share of the result is
// divided by 16, so there it does not matter (with n0 a subnormal too, scores were off by 1e-5).
// BASE: the fp16 number whose mantissa takes n0: 0x6400 (1024) gives n0, 0x2c00 gives n0 * 2^-14.
template <uint32_t BASE>
struct U4Word {
  uint32_t a_u, b_u, a_n, b_n;
  __device__ __forceinline__ explicit U4Word(uint32_t w) {
    constexpr uint32_t base = BASE * 0x10001u;
    a_u = w & 0x00ff00ffu;
    b_u = __byte_perm(w, 0u, 0x4341);
    a_n = hsub2_u32(and_or(w, 0x000f000fu, base), base);
    b_n = hsub2_u32(and_or(b_u, 0x000f000fu, base), base);
  }
};

// Launch shape by head size; registers and shared memory are split evenly among the resident blocks.
template <int HD>
struct U4Shape;
template <int W, int B, int P, int N, int C>
struct U4ShapeOf {
  static constexpr int WARPS = W;    // of a block
  static constexpr int BLOCKS = B;   // resident per SM
  static constexpr int PAGES = P;    // a warp works on at once
  static constexpr int SLOTS = N, CLUSTER_SLOTS = C;    // stages of a warp, a multiple of PAGES
};
template <>
struct U4Shape<64> : U4ShapeOf<4, 4, 2, 8, 4> {};
template <>
struct U4Shape<128> : U4ShapeOf<4, 3, 2, 6, 4> {};
template <>
struct U4Shape<256> : U4ShapeOf<4, 2, 1, 4, 4> {};
constexpr float U4_LIMIT = 14.9f;   // p'' <= 2^14.9, and p'' f below the largest fp16 number
constexpr float U4_LEVEL = 9.0f;    // p'' of the largest z when the reference moves
constexpr float U4_SPREAD = 16.0f;  // a class of rows: powers of two down to 1 / 16 of its largest
constexpr float U4_REACH = 0x1p90f; // how far below the widest class yet a reference follows: outputs scaled up by it still fit f32

// CLUSTER: the instance whose splits merge through distributed shared memory needs room to receive; the other gives that
// room to the ring.
template <int HD, bool CLUSTER>
struct U4Smem {
  static constexpr int G = HD / QGROUP;
  static constexpr int STEPS = PAGE_TOKENS * HD / 2;          // 2 bytes per (row, group)
  static constexpr int BIASES = STEPS + PAGE_TOKENS * G * 2;  // bf16 [row][group]
  static constexpr int POWERS = BIASES + PAGE_TOKENS * G * 2; // 8 x bf16
  static constexpr int TILE = POWERS + 16;
  static constexpr int STAGE = 2 * TILE;
  static constexpr int SLOTS = CLUSTER ? U4Shape<HD>::CLUSTER_SLOTS : U4Shape<HD>::SLOTS, WARPS = U4Shape<HD>::WARPS, THREADS = WARPS * 32;
  static constexpr int OPAD = HD + 4;
  static constexpr int Q_BYTES = G * 2 * 32 * 16;             // B fragments: [group][high | low dims][lane]{hi, lo}
  static constexpr int QROWS_BYTES = 8 * HD * 4;              // q in f32 while the fragments are made
  static constexpr int QSUM_BYTES = 8 * 8 * 4 + 8 * 4;        // [head][8 groups], absent groups zero; power of two per head
  static constexpr int O_BYTES = WARPS * 8 * OPAD * 4;
  static constexpr int ML_BYTES = (WARPS * 24 + 16) * 4;   // what finish_block asks for
  static constexpr int BAR_BYTES = (WARPS * SLOTS * 8 + 15) / 16 * 16;
  // the row of a fused append: f32 K and V, afterwards its bytes (codes K | V, then 4 G + 1 half words)
  static constexpr int NEW_BYTES = 2 * HD * 4;
  static constexpr int RECV_BYTES = CLUSTER ? ClusterRecv<HD>::BYTES : 0;
  static constexpr int FIXED = Q_BYTES + QROWS_BYTES + QSUM_BYTES + ML_BYTES + BAR_BYTES + 64 + NEW_BYTES + RECV_BYTES;
  static constexpr int RING_BYTES = WARPS * SLOTS * STAGE > O_BYTES ? WARPS * SLOTS * STAGE : O_BYTES;
  static constexpr int TOTAL = RING_BYTES + FIXED;
  static_assert(U4_EXP_MIN == -40, "the largest 2^-e of a row is 2^40");
  static_assert(STAGE % 16 == 0 && TILE % 16 == 0 && QSUM_BYTES % 16 == 0, "16-byte pieces");
  static_assert(RING_BYTES % 16 == 0 && BAR_BYTES % 16 == 0, "16-byte pieces");
};

// N words from shared memory with loads as wide as N words.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
    }
  }
}

// Writes the row that a fused append has quantised (`park`) into a tile pair in global or shared memory; one warp.
template <int HD>
__device__ __forceinline__ void u4_place_row(uint8_t* ktile, const uint8_t* park, int rin, int lane) {
  using S = U4Smem<HD, false>;
  uint8_t* vtile = ktile + S::TILE;
  const uint16_t* meta = reinterpret_cast<const uint16_t*>(park + HD);   // K step, K bias, V factor, V bias [G] each, power
  const int p = lane & 15;
#pragma unroll
  for (int grp = 0; grp < S::G; ++grp) {
    const int dim = grp * QGROUP + p;
    if (lane < 16) ktile[u4_k_byte(rin, dim, HD)] = park[grp * 16 + p];
    else vtile[u4_v_byte(rin, dim, HD)] = park[HD / 2 + grp * 16 + p];
  }
  if (lane < S::G) {
    *reinterpret_cast<uint16_t*>(ktile + u4_step_offset(0, rin, lane, HD)) = meta[lane];
    *reinterpret_cast<uint16_t*>(ktile + u4_bias_offset(rin, lane, HD)) = meta[S::G + lane];
    *reinterpret_cast<uint16_t*>(vtile + u4_step_offset(1, rin, lane, HD)) = meta[2 * S::G + lane];
    *reinterpret_cast<uint16_t*>(vtile + u4_bias_offset(rin, lane, HD)) = meta[3 * S::G + lane];
  }
  if (lane == 0) *reinterpret_cast<uint16_t*>((rin < 8 ? ktile : vtile) + u4_pow_offset(rin, HD)) = meta[4 * S::G];
}

// PP: pages a warp works on at once. Two (head_dim 128) give the chains of matrix instructions twice the
// independent work and share the query's fragments and the bookkeeping; with head_dim 256 one page fills the registers.
// PAIRED (up to four query heads per KV head): the matrix instruction has eight columns, so column h + 4 takes the lo parts
// of head h's query and weights beside the hi parts in column h: half the products and half their chains (32/8 heads of 128: 24
// uneven sequences 47.0 -> 42.5 us, 16 of 12000 rows 74.2 -> 67.3).
// (Even batches place two blocks per SM: the cluster instance, which only they use, is compiled for no more than that. At three
// it spilled, and 8 sequences of 32768 rows, 32/4 heads of 128, took 54.2 us instead of 51.6.)
template <int HD, bool CLUSTER, bool PEERS, bool PAIRED>
__global__ void __launch_bounds__(U4Shape<HD>::WARPS * 32, CLUSTER && U4Shape<HD>::BLOCKS == 3 ? 2 : U4Shape<HD>::BLOCKS)
    attention_u4_kernel(AttnArgs a) {
  using S = U4Smem<HD, CLUSTER>;
  constexpr int G = S::G;
  constexpr int PP = U4Shape<HD>::PAGES, WARPS = S::WARPS, THREADS = S::THREADS;
  constexpr int GS = G < 4 ? G : 4, SETS = G / GS;   // groups whose products are formed side by side
  // (not rounded up by hand: an address that went through an integer is a generic one to the compiler, and its loads too)
  extern __shared__ __align__(128) uint8_t u4_smem[];
  uint8_t* ring = u4_smem;
  uint8_t* q_frag = ring + S::RING_BYTES;
  float* q_rows = reinterpret_cast<float*>(q_frag + S::Q_BYTES);          // [8][HD]
  float* qsum_s = q_rows + 8 * HD;                                        // [8][8]
  float* qpow_s = qsum_s + 64;                                            // [8]
  float* o_s = reinterpret_cast<float*>(ring);    // aliases the ring once it has drained
  float* ml_s = qpow_s + 8;                                               // [warps][8][2]
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(ml_s) + S::ML_BYTES);
  int* flags = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + S::BAR_BYTES);
  float* new_s = reinterpret_cast<float*>(flags + 16);
  float* recv_s = new_s + 2 * HD;
  volatile int* abort_flag = flags;

  const int split = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);   // uniform over the warp, and known to be
  const int gqa = a.q_heads / a.pool.kv_heads;
  const int slot = a.slots ? a.slots[seq] : a.slot0;
  int32_t* len_ptr = a.pool.lens + int64_t(slot) * a.pool.layers + a.layer;
  const bool do_append = a.k_new != nullptr;
  if (a.pdl_trigger) pdl_launch_dependents();

  const int len_old = *reinterpret_cast<const volatile int32_t*>(len_ptr);
  const int len = len_old + (do_append ? 1 : 0);
  int64_t start = a.sliding_window > 0 ? (len > a.sliding_window ? len - a.sliding_window : 0) : a.window_start;
  if (start >= len) start = len > 0 ? len - 1 : 0;
  const int ws = static_cast<int>(start);
  const int sinks = static_cast<int>(a.sink_rows < ws ? a.sink_rows : ws);   // rows [0, sinks) and [ws, len) are seen
  const int p_first = ws / PAGE_TOKENS;
  const int sink_pages = min((sinks + PAGE_TOKENS - 1) / PAGE_TOKENS, p_first);
  const PageMap map{sink_pages, p_first - sink_pages};
  const int n_pages = sink_pages + (len - 1) / PAGE_TOKENS - p_first + 1;
  int splits = a.splits;
  if (a.pages_per_split > 0) {
    const int want = (n_pages + a.pages_per_split - 1) / a.pages_per_split;
    splits = want < 1 ? 1 : min(want, a.splits);
  }
  if (split >= splits) return;
  const int pb = static_cast<int>(int64_t(n_pages) * split / splits);
  const int pe = static_cast<int>(int64_t(n_pages) * (split + 1) / splits);
  const int my_pages = pe - pb;
  const int32_t* table = a.pool.tables + int64_t(slot) * a.pool.table_stride;
  const int64_t head_off = int64_t(a.layer) * a.pool.layer_bytes + int64_t(kvh) * 2 * a.pool.tile_bytes;
  const bool owns_append = do_append && pe == n_pages && my_pages > 0;   // the new row lies in the last page

  // Every warp owns SLOTS neighbouring stages of the ring and fetches its own pages: its n-th page has ordinal pb + warp + 4 n
  // and goes to its stage n % SLOTS, one bulk copy per page, completion on the stage's barrier. A stage is refilled by the
  // warp itself as soon as it has used it up, so no second barrier and no producer stand between the two (a producer warp
  // needed about 640 cycles per page, waiting for the consumers' releases one by one).
  // Lane l holds the block-table entries of the warp's pages 32 k + l: batch k and the one after it.
  constexpr int SLOTS = S::SLOTS;
  const int count = (my_pages - warp + WARPS - 1) / WARPS;   // this warp's pages
  const auto entry_of = [&](int n) {
    int32_t page = 0;
    if (n < count) {
      page = table[map.page(pb + warp + WARPS * n)];
      if (page < 0 || page >= a.num_pages) {   // reported; the page read in its place is one of the pool's
        atomicExch(a.status, DEV_ERR_BAD_PAGE);
        page = 0;
      }
    }
    return page;
  };
  int32_t entries = entry_of(lane), entries_next = entry_of(32 + lane);
  const uint8_t* my_ring = ring + warp * SLOTS * S::STAGE;
  const uint32_t my_ring_at = smem_u32(my_ring), my_bars = smem_u32(bars + warp * SLOTS);
  const uint64_t policy = l2_policy_evict_first();
  const uint8_t* const source = a.pool.base + head_off;
  const int64_t page_bytes = a.pool.page_bytes;
  const auto fetch = [&](int slot_at, int32_t page) {   // one lane
    const uint32_t bar = my_bars + 8 * slot_at;
    mbar_expect_tx(bar, S::STAGE);
    bulk_copy_g2s(my_ring_at + slot_at * S::STAGE, source + page * page_bytes, S::STAGE, bar, policy);
  };
  if (tid == 0) {
    flags[0] = 0;   // a wait ran out
    flags[1] = 0;
    flags[5] = 0;   // set once the quantised row of a fused append is parked in shared memory
  }
  if (lane < SLOTS) mbar_init(my_bars + 8 * lane, 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  if (lane < SLOTS && lane < count) fetch(lane, entries);
  {
    // ---------------- the query ----------------
    constexpr int NV = (8 * HD / 4 + THREADS - 1) / THREADS;   // 16-byte pieces of q per thread
    const float* q = a.q + (int64_t(seq) * a.q_heads + int64_t(kvh) * gqa) * HD;
    // q and the row to append come from the launch before this one; the cursor, the block table and
    // the pages the producer starts to copy do not
    if (a.pdl_wait) pdl_wait();
    float4 v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int f = (tid + k * THREADS) * 4;
      v[k] = (f / HD < gqa) ? __ldg(reinterpret_cast<const float4*>(q + f)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (owns_append && tid * 4 < 2 * HD) {
      const int64_t row_off = int64_t(seq) * a.pool.kv_heads * HD + kvh * HD;
      const float* src = tid * 4 < HD ? a.k_new + row_off + tid * 4 : a.v_new + row_off + (tid * 4 - HD);
      *reinterpret_cast<float4*>(new_s + tid * 4) = __ldg(reinterpret_cast<const float4*>(src));
    }
    if (owns_append && tid == 0) flags[2] = table[len_old / PAGE_TOKENS];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int f = (tid + k * THREADS) * 4;
      v[k].x *= a.scale_log2e, v[k].y *= a.scale_log2e, v[k].z *= a.scale_log2e, v[k].w *= a.scale_log2e;
      if (f < 8 * HD) *reinterpret_cast<float4*>(q_rows + f) = v[k];
    }
    __syncthreads();
    // The power of two that brings the largest |q| of a head to 2^15..2^16.
#pragma unroll
    for (int h = warp; h < 8; h += WARPS) {
      float big = 0.0f;
#pragma unroll
      for (int grp = 0; grp < G; ++grp) big = fmaxf(big, fabsf(q_rows[h * HD + grp * QGROUP + lane]));
      asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(big) : "f"(big));
      if (lane == 0) {
        const int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
        qpow_s[h] = pow2f(max(-90, min(90, e - 15)));   // q = qpow * (what the fragments hold)
      }
      if (G < 8 && lane >= G && lane < 8) qsum_s[h * 8 + lane] = 0.0f;
    }
    __syncthreads();
    for (int i = tid; i < G * 32; i += THREADS) {
      const int grp = i >> 5, column = (i & 31) >> 2, t = i & 3;
      const int h = PAIRED ? column & 3 : column;
      const float inv = 1.0f / qpow_s[h];
      const float* row = q_rows + h * HD + grp * QGROUP + 4 * t;
      const float4 x = *reinterpret_cast<const float4*>(row), y = *reinterpret_cast<const float4*>(row + 16);
      // the group's sum, over the four threads that hold it
      float sum = (x.x + x.y) + (x.z + x.w) + ((y.x + y.y) + (y.z + y.w));
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == 0) qsum_s[column * 8 + grp] = PAIRED && column > 3 ? 0.0f : sum;
      // n0 x + n1 y = n0 (x - y / 16) + u (y / 16), with u in units of 2^-24 and n0 in units of 2^-14
      const float s = inv * 0.0625f, d = 0x1p-10f;
      const float u[4] = {y.x * s, y.y * s, y.z * s, y.w * s};
      const float r[4] = {fmaf(x.x, inv, -u[0]) * d, fmaf(x.y, inv, -u[1]) * d, fmaf(x.z, inv, -u[2]) * d, fmaf(x.w, inv, -u[3]) * d};
      // k-slots (2t, 2t+1) are the bytes 0 and 2 of a word, (2t+8, 2t+9) the bytes 1 and 3
      uint4 fu, fr;
      fu.x = pack_f16(u[0], u[2]), fu.y = pack_f16(u[1], u[3]);
      fr.x = pack_f16(r[0], r[2]), fr.y = pack_f16(r[1], r[3]);
      const float2 u0 = unpack_f16(fu.x), u1 = unpack_f16(fu.y), r0 = unpack_f16(fr.x), r1 = unpack_f16(fr.y);
      fu.z = pack_f16(u[0] - u0.x, u[2] - u0.y), fu.w = pack_f16(u[1] - u1.x, u[3] - u1.y);
      fr.z = pack_f16(r[0] - r0.x, r[2] - r0.y), fr.w = pack_f16(r[1] - r1.x, r[3] - r1.y);
      if (PAIRED) {
        *reinterpret_cast<uint4*>(q_frag + i * 16) = column < 4 ? make_uint4(fu.x, fu.y, fr.x, fr.y) : make_uint4(fu.z, fu.w, fr.z, fr.w);
      } else {
        *reinterpret_cast<uint4*>(q_frag + ((grp * 2) * 32 + (i & 31)) * 16) = fu;
        *reinterpret_cast<uint4*>(q_frag + ((grp * 2 + 1) * 32 + (i & 31)) * 16) = fr;
      }
    }
    __syncthreads();   // fragments and sums written
    // The bias product's B fragment: group sums as three bf16 parts. With two groups the sixteen k-slots take
    // {hi, mid, lo, nothing x 5}, with four {hi, mid, lo, nothing}; with eight, {hi, mid}, and lo goes through a k = 8 product.
    uint32_t qs0, qs1, qs2 = 0;
    {
      const int g = lane >> 2, t = lane & 3;
      const int pair = G == 2 ? 0 : G == 4 ? (t & 1) : t;
      const float2 x = *reinterpret_cast<const float2*>(qsum_s + g * 8 + 2 * pair);
      const uint32_t hi = pack_bf16(x.x, x.y);
      const float2 r = make_float2(x.x - bf16_lo_f32(hi), x.y - bf16_hi_f32(hi));
      const uint32_t mid = pack_bf16(r.x, r.y);
      const uint32_t lo = pack_bf16(r.x - bf16_lo_f32(mid), r.y - bf16_hi_f32(mid));
      if (G == 2) qs0 = t == 0 ? hi : t == 1 ? mid : t == 2 ? lo : 0u, qs1 = 0u;
      else if (G == 4) qs0 = t < 2 ? hi : mid, qs1 = t < 2 ? lo : 0u;
      else qs0 = hi, qs1 = mid, qs2 = lo;
    }
    const int g = lane >> 2, t = lane & 3;
    const int h0 = PAIRED ? 2 * (t & 1) : 2 * t;   // this thread's heads: h0 and h0 + 1
    const float ch0 = qpow_s[h0] * 16777216.0f, ch1 = qpow_s[h0 + 1] * 16777216.0f;   // products are in units of 2^-24
    const float once = PAIRED && t > 1 ? 0.0f : 1.0f;             // what is added to a score once: in the hi column
    const uint32_t low = PAIRED && g < 4 ? 0u : 0xffffffffu;      // PAIRED: column g takes lo parts

    // The row of a fused append is quantised now, by the warp with the fewest pages, while the first pages are
    // on their way; its bytes go to the page in global memory and stay parked in shared memory for the warp
    // that will meet the page in the ring.
    uint8_t* park = reinterpret_cast<uint8_t*>(new_s);
    if (owns_append && warp == WARPS - 1) {
      const int rin = len_old % PAGE_TOKENS;
      const uint32_t odd = rin & 1;
      const int32_t page = flags[2];
      float x[2 * G];
#pragma unroll
      for (int i = 0; i < 2 * G; ++i) x[i] = new_s[i * QGROUP + lane];
      __syncwarp();
      uint32_t code[2 * G];
      uint16_t* meta = reinterpret_cast<uint16_t*>(park + HD);
#pragma unroll
      for (int is_v = 0; is_v < 2; ++is_v) {
        U4Row<G> row;
        row.quantize(*reinterpret_cast<float(*)[G]>(x + is_v * G), odd);
#pragma unroll
        for (int grp = 0; grp < G; ++grp) {
          code[is_v * G + grp] = row.code[grp];
          if (lane == grp) {
            meta[is_v * 2 * G + grp] = is_v ? u4_v_factor_bits(row.step[grp], row.exponent, odd) : static_cast<uint16_t>(row.step[grp] ^ (odd << 15));
            meta[is_v * 2 * G + G + grp] = row.bias[grp];
          }
        }
        if (is_v && lane == 0) meta[4 * G] = static_cast<uint16_t>(__float_as_uint(pow2f(row.exponent)) >> 16);
      }
#pragma unroll
      for (int grp = 0; grp < G; ++grp) {
        // lanes 0-15 put the K byte together, lanes 16-31 the V byte
        const uint32_t other = __shfl_xor_sync(0xffffffffu, lane < 16 ? code[G + grp] : code[grp], 16);
        park[(lane < 16 ? 0 : HD / 2) + grp * 16 + (lane & 15)] =
            static_cast<uint8_t>(lane < 16 ? code[grp] | (other << 4) : other | (code[G + grp] << 4));
      }
      __syncwarp();
      // a bad table entry is reported where the page is fetched
      if (page >= 0 && page < a.num_pages) u4_place_row<HD>(a.pool.base + int64_t(page) * a.pool.page_bytes + head_off, park, rin, lane);
      __syncwarp();
      if (lane == 0) {
        __threadfence_block();
        *reinterpret_cast<volatile int*>(flags + 5) = 1;
      }
    }

    // ---------------- the pages ----------------
    float o_hi[G][4], o_lo[G][4], o_b[2][G];   // o_b: V biases, [head 2t, 2t + 1][group]
#pragma unroll
    for (int grp = 0; grp < G; ++grp) {
      o_hi[grp][0] = o_hi[grp][1] = o_hi[grp][2] = o_hi[grp][3] = 0.0f;
      o_lo[grp][0] = o_lo[grp][1] = o_lo[grp][2] = o_lo[grp][3] = 0.0f;
      o_b[0][grp] = o_b[1][grp] = 0.0f;
    }
    float top0 = -1.0e30f, top1 = -1.0e30f;   // m0, m1 + U4_LIMIT
    float m0 = -1.0e30f, m1 = -1.0e30f, l0 = 0.0f, l1 = 0.0f;
    // The references are for rows with 2^-e <= back_limit (0: for none yet). While an iteration's rows are worked on class by class
    // back_limit is negative, and rows with 2^-e <= taken are done.
    float back_limit = 0.0f, taken = 0.0f, widest = INFINITY;   // widest: the least back_limit so far
    const int k_off = g * (HD / 2) + t * (HD == 64 ? 4 : 16);                 // + (set ^ odd row) * 64; row g + 8: + 4 * HD
    const int kb_off = S::BIASES + g * G * 2 + (G == 2 ? 0 : G == 4 ? (t & 1) : t) * 4;    // K biases of row g
    const int vs_off = S::TILE + S::STEPS + t * G * 4;                        // V factors of rows 2t, 2t+1; rows + 8: + 16 * G
    const int vb_off = S::TILE + S::BIASES + g * G * 2;                       // V biases of row g; row g + 8: + 16 * G
    // Iterations that are not like the others: a page is not seen whole (the last of the sinks, the window's first, the
    // last), takes the appended row, or is missing because the warp's pages are an odd number.
    const auto next_special = [&](int from) {
      int best = INT32_MAX;
      const auto consider = [&](int v) {   // ordinal of a page
        const int k = v - pb - warp;
        if (k >= 0 && k % WARPS == 0 && k / WARPS < count) {
          const int at = k / WARPS / PP * PP;
          if (at >= from) best = min(best, at);
        }
      };
      if (sinks % PAGE_TOKENS) consider(sink_pages - 1);
      if (ws % PAGE_TOKENS) consider(sink_pages);
      if (len % PAGE_TOKENS || do_append) consider(n_pages - 1);
      if (count % PP && count - count % PP >= from) best = min(best, count - count % PP);
      return best;
    };
    int special_at = next_special(0);
    int at = 0, phase = 0;   // stage of the iteration's first page
    int batch = 0;           // first page of the entries held
    for (int n = 0; n < count; n += PP) {
      const uint8_t* tile[PP];
      bool ok = true, again = false;
      // (a missing second page stands in for itself by the first one)
#pragma unroll
      for (int u = 0; u < PP; ++u) tile[u] = my_ring + (at + (u > 0 && n + u >= count ? 0 : u)) * S::STAGE;
      {
        const uint32_t bar = my_bars + 8 * at;
        const bool pair = PP > 1 && n + 1 < count;
        bool ready = mbar_try_wait(bar, phase);
        if (PP > 1) ready = (mbar_try_wait(bar + (pair ? 8 : 0), phase)) && ready;
        if (__any_sync(0xffffffffu, !ready))
          ok = mbar_wait_warp(bar, phase, abort_flag, a.status) && mbar_wait_warp(bar + (pair ? 8 : 0), phase, abort_flag, a.status);
      }
      if (!ok) {
        // gave up (reported): the copies still on their way are waited for, with the short bound, before the block leaves
        for (int k = n; k < count && k < n + SLOTS; ++k) {
          int slot_at = at + (k - n), ph = phase;
          if (slot_at >= SLOTS) slot_at -= SLOTS, ph ^= 1;
          mbar_wait(my_bars + 8 * slot_at, ph, abort_flag, a.status);
        }
        break;
      }
      const bool special = n == special_at;
      if (special) {
        special_at = next_special(n + PP);
        const int k = n_pages - 1 - pb - warp - n * WARPS;   // the last page is the iteration's page k / 4
        if (owns_append && k >= 0 && k < PP * WARPS && k % WARPS == 0) {
          // the new row joins the staged copy
          uint32_t spins = 0;
          while (*reinterpret_cast<volatile int*>(flags + 5) == 0) {
            if (++spins > WAIT_SPINS) {
              *abort_flag = 1;
              atomicExch(a.status, DEV_ERR_WAIT_TIMEOUT);
              break;
            }
          }
          __syncwarp();
          u4_place_row<HD>(ring + (warp * SLOTS + at + k / WARPS) * S::STAGE, park, len_old % PAGE_TOKENS, lane);
          __syncwarp();
        }
      }
      {
        // ---- scores ----
        float z[PP][4];   // (row g; heads 2t, 2t+1), (row g + 8; ...)
        float acc[PP][GS][4];
#pragma unroll
        for (int u = 0; u < PP; ++u) z[u][0] = z[u][1] = z[u][2] = z[u][3] = 0.0f;
#pragma unroll
        for (int set = 0; set < SETS; ++set) {
          uint32_t w0[PP][GS], w1[PP][GS];   // codes of rows g and g + 8
#pragma unroll
          for (int u = 0; u < PP; ++u) {
            const uint8_t* at = tile[u] + k_off + (SETS > 1 ? (set ^ (g & 1)) : 0) * 64;
            if constexpr (HD == 64) {
              w0[u][0] = *reinterpret_cast<const uint32_t*>(at), w0[u][1] = *reinterpret_cast<const uint32_t*>(at + 16);
              w1[u][0] = *reinterpret_cast<const uint32_t*>(at + 4 * HD), w1[u][1] = *reinterpret_cast<const uint32_t*>(at + 4 * HD + 16);
            } else {
              load_words<GS>(at, w0[u]);
              load_words<GS>(at + 4 * HD, w1[u]);
            }
          }
#pragma unroll
          for (int j = 0; j < GS; ++j) {
            uint4 fu, fr;
            if (PAIRED) {
              fu = *reinterpret_cast<const uint4*>(q_frag + ((set * 4 + j) * 32 + lane) * 16);
              fr = make_uint4(fu.z, fu.w, 0u, 0u);
            } else {
              fu = *reinterpret_cast<const uint4*>(q_frag + (((set * 4 + j) * 2) * 32 + lane) * 16);
              fr = *reinterpret_cast<const uint4*>(q_frag + (((set * 4 + j) * 2 + 1) * 32 + lane) * 16);
            }
#pragma unroll
            for (int u = 0; u < PP; ++u) {
              const U4Word<0x2c00> c0(w0[u][j]), c1(w1[u][j]);
              if (PAIRED) {
                mma_f16_zero(acc[u][j], c0.a_n, c1.a_n, c0.b_n, c1.b_n, fr.x, fr.y);
              } else {
                mma_f16_zero(acc[u][j], c0.a_u, c1.a_u, c0.b_u, c1.b_u, fu.z, fu.w);   // the small parts first: the
                mma_f16(acc[u][j], c0.a_n, c1.a_n, c0.b_n, c1.b_n, fr.z, fr.w);   // accumulator is truncated after
                mma_f16(acc[u][j], c0.a_n, c1.a_n, c0.b_n, c1.b_n, fr.x, fr.y);   // every product
              }
              mma_f16(acc[u][j], c0.a_u, c1.a_u, c0.b_u, c1.b_u, fu.x, fu.y);
            }
          }
#pragma unroll
          for (int u = 0; u < PP; ++u) {
            uint32_t s0[GS / 2], s1[GS / 2];
            load_words<GS / 2>(tile[u] + S::STEPS + g * G * 2 + set * 8, s0);
            load_words<GS / 2>(tile[u] + S::STEPS + (g + 8) * G * 2 + set * 8, s1);
#pragma unroll
            for (int j = 0; j < GS; ++j) {
              const float a0 = j & 1 ? bf16_hi_f32(s0[j >> 1]) : bf16_lo_f32(s0[j >> 1]);
              const float a1 = j & 1 ? bf16_hi_f32(s1[j >> 1]) : bf16_lo_f32(s1[j >> 1]);
              z[u][0] = fmaf(a0, acc[u][j][0], z[u][0]);
              z[u][1] = fmaf(a0, acc[u][j][1], z[u][1]);
              z[u][2] = fmaf(a1, acc[u][j][2], z[u][2]);
              z[u][3] = fmaf(a1, acc[u][j][3], z[u][3]);
            }
          }
        }
        float back[PP][2];   // 2^-e of rows g, g + 8
        bool over = false;
#pragma unroll
        for (int u = 0; u < PP; ++u) {
          const uint32_t e0 = *reinterpret_cast<const uint16_t*>(tile[u] + S::POWERS + 2 * g);
          const uint32_t e1 = *reinterpret_cast<const uint16_t*>(tile[u] + S::TILE + S::POWERS + 2 * g);
          back[u][0] = __uint_as_float(0x7f000000u - (e0 << 16));
          back[u][1] = __uint_as_float(0x7f000000u - (e1 << 16));
          const float x0 = fmaf(__uint_as_float(0x4b000000u | (e0 >> 7)), once, -8388735.0f * once);   // e = exponent field - 127
          const float x1 = fmaf(__uint_as_float(0x4b000000u | (e1 >> 7)), once, -8388735.0f * once);
          float sb[4] = {x0, x0, x1, x1};
          const uint32_t b0 = *reinterpret_cast<const uint32_t*>(tile[u] + kb_off);
          const uint32_t b1 = *reinterpret_cast<const uint32_t*>(tile[u] + kb_off + 16 * G);
          mma_bf16(sb, b0, b1, b0, b1, qs0, qs1);
          if (G == 8) mma_bf16_k8(sb, b0, b1, qs2);
          fma2(sb[0], sb[1], z[u][0], z[u][1], ch0, ch1);
          fma2(sb[2], sb[3], z[u][2], z[u][3], ch0, ch1);
          if (PAIRED) {   // hi and lo columns
            const float other[4] = {__shfl_xor_sync(0xffffffffu, sb[0], 2), __shfl_xor_sync(0xffffffffu, sb[1], 2),
                                    __shfl_xor_sync(0xffffffffu, sb[2], 2), __shfl_xor_sync(0xffffffffu, sb[3], 2)};
            add2(sb[0], sb[1], other[0], other[1]);
            add2(sb[2], sb[3], other[2], other[3]);
          }
          z[u][0] = sb[0], z[u][1] = sb[1], z[u][2] = sb[2], z[u][3] = sb[3];
        }
        uint32_t vs0[PP][G], vs1[PP][G];           // V factors of the groups: rows (2t, 2t+1) and (2t+8, 2t+9)
        uint32_t vb0[PP][G / 2], vb1[PP][G / 2];   // V biases, two groups a word: rows g and g + 8
#pragma unroll
        for (int u = 0; u < PP; ++u) {
          load_words<G>(tile[u] + vs_off, vs0[u]);
          load_words<G>(tile[u] + vs_off + 16 * G, vs1[u]);
          load_words<G / 2>(tile[u] + vb_off, vb0[u]);
          load_words<G / 2>(tile[u] + vb_off + 16 * G, vb1[u]);
        }
        if (special) {
          // A row that is not seen weighs nothing, whatever its bytes say.
#pragma unroll
          for (int u = 0; u < PP; ++u) {
            const int v = pb + warp + WARPS * (n + u);
            const int base = u == 0 || n + u < count ? (v + (v >= sink_pages ? p_first - sink_pages : 0)) * PAGE_TOKENS : len;
            const auto seen = [&](int r) {
              const int row = base + r;
              return row < len && (row < sinks || row >= ws);
            };
            const bool s0 = seen(g), s1 = seen(g + 8);
            if (!s0) z[u][0] = z[u][1] = -INFINITY, back[u][0] = 0.0f;
            if (!s1) z[u][2] = z[u][3] = -INFINITY, back[u][1] = 0.0f;
            const uint32_t k0 = (seen(2 * t) ? 0x0000ffffu : 0u) | (seen(2 * t + 1) ? 0xffff0000u : 0u);
            const uint32_t k1 = (seen(2 * t + 8) ? 0x0000ffffu : 0u) | (seen(2 * t + 9) ? 0xffff0000u : 0u);
#pragma unroll
            for (int grp = 0; grp < G; ++grp) vs0[u][grp] &= k0, vs1[u][grp] &= k1;
#pragma unroll
            for (int i = 0; i < G / 2; ++i) vb0[u][i] = s0 ? vb0[u][i] : 0u, vb1[u][i] = s1 ? vb1[u][i] : 0u;
          }
        }
        float mx0 = fmaxf(z[0][0], z[0][2]), mx1 = fmaxf(z[0][1], z[0][3]), most_back = fmaxf(back[0][0], back[0][1]);
        if (PP == 2) {
          mx0 = fmaxf(mx0, fmaxf(z[PP - 1][0], z[PP - 1][2])), mx1 = fmaxf(mx1, fmaxf(z[PP - 1][1], z[PP - 1][3]));
          most_back = fmaxf(most_back, fmaxf(back[PP - 1][0], back[PP - 1][1]));
        }
        over = mx0 > top0 || mx1 > top1 || most_back > back_limit;
        if (__any_sync(0xffffffffu, over)) {
          // The class of this pass: the rows left with the largest powers of two, down to 1 / U4_SPREAD of the largest.
          float least = INFINITY;
#pragma unroll
          for (int u = 0; u < PP; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              if (back[u][r] > 0x1p40f) {   // a row that nobody wrote: zeros, its e read as -127, which becomes the least there is
                z[u][2 * r] += 127 + U4_EXP_MIN, z[u][2 * r + 1] += 127 + U4_EXP_MIN;
                back[u][r] = 0x1p40f;
              }
              if (back[u][r] > taken) least = fminf(least, back[u][r]);
            }
          asm("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(least) : "f"(least));
          const float limit = least * U4_SPREAD;
          bool left = false;
#pragma unroll
          for (int u = 0; u < PP; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              left = left || back[u][r] > limit;
              if (back[u][r] > limit || back[u][r] <= taken) z[u][2 * r] = z[u][2 * r + 1] = -INFINITY, back[u][r] = 0.0f;
            }
          again = __any_sync(0xffffffffu, left);
          // Its references: the ones there are, moved by the distance of the classes in powers of two, so that a row's p'' goes by
          // its share in the sum of the weights, whatever class it is of; raised below where a score asks for it.
          const float ref = fminf(limit, widest * U4_REACH);
          widest = fminf(widest, limit);
          const float shift = static_cast<float>((__float_as_int(fabsf(back_limit)) - __float_as_int(ref)) >> 23);
          taken = again ? limit : 0.0f;
          back_limit = again ? -ref : ref;
          mx0 = fmaxf(z[0][0], z[0][2]), mx1 = fmaxf(z[0][1], z[0][3]);
          if (PP == 2) mx0 = fmaxf(mx0, fmaxf(z[PP - 1][0], z[PP - 1][2])), mx1 = fmaxf(mx1, fmaxf(z[PP - 1][1], z[PP - 1][3]));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
          }
          float mn0 = m0 + shift, mn1 = m1 + shift;
          if (mx0 > mn0 + U4_LIMIT) mn0 = floorf(mx0 - U4_LEVEL);   // whole numbers: what is scaled below loses nothing
          if (mx1 > mn1 + U4_LIMIT) mn1 = floorf(mx1 - U4_LEVEL);
          const float al0 = exp2f(m0 - mn0), al1 = exp2f(m1 - mn1);
          l0 *= al0;
          l1 *= al1;
#pragma unroll
          for (int grp = 0; grp < G; ++grp) {
            o_hi[grp][0] *= al0, o_hi[grp][2] *= al0, o_lo[grp][0] *= al0, o_lo[grp][2] *= al0, o_b[0][grp] *= al0;
            o_hi[grp][1] *= al1, o_hi[grp][3] *= al1, o_lo[grp][1] *= al1, o_lo[grp][3] *= al1, o_b[1][grp] *= al1;
          }
          m0 = mn0;
          m1 = mn1;
          top0 = mn0 + U4_LIMIT, top1 = mn1 + U4_LIMIT;
        }
        // ---- weights ----
        uint32_t ph[PP][2], pl[PP][2];
#pragma unroll
        for (int u = 0; u < PP; ++u) {
          add2(z[u][0], z[u][1], -m0, -m1);
          add2(z[u][2], z[u][3], -m0, -m1);
          float p[4] = {exp2_ftz(z[u][0]), exp2_ftz(z[u][1]), exp2_ftz(z[u][2]), exp2_ftz(z[u][3])};
          const uint32_t h0 = pack_f16(p[0], p[1]), h1 = pack_f16(p[2], p[3]);
          const float2 f0 = unpack_f16(h0), f1 = unpack_f16(h1);
          float d[4] = {p[0], p[1], p[2], p[3]};
          add2(d[0], d[1], -f0.x, -f0.y);
          add2(d[2], d[3], -f1.x, -f1.y);
          const uint32_t d0 = pack_f16(d[0], d[1]), d1 = pack_f16(d[2], d[3]);
          // (row g; heads 2t, 2t+1) -> (rows 2t, 2t+1; head g)
          ph[u][0] = movmatrix_trans(h0), ph[u][1] = movmatrix_trans(h1);
          pl[u][0] = movmatrix_trans(d0), pl[u][1] = movmatrix_trans(d1);
          mul2(p[0], p[1], back[u][0], back[u][0]);
          mul2(p[2], p[3], back[u][1], back[u][1]);
          add2(l0, l1, p[0], p[1]);
          add2(l0, l1, p[2], p[3]);
#pragma unroll
          for (int i = 0; i < G / 2; ++i) {
            const float b0[2] = {bf16_lo_f32(vb0[u][i]), bf16_hi_f32(vb0[u][i])}, b1[2] = {bf16_lo_f32(vb1[u][i]), bf16_hi_f32(vb1[u][i])};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              fma2(o_b[h][2 * i], o_b[h][2 * i + 1], b0[0], b0[1], p[h], p[h]);
              fma2(o_b[h][2 * i], o_b[h][2 * i + 1], b1[0], b1[1], p[2 + h], p[2 + h]);
            }
          }
        }
        // ---- outputs. The matrix instruction truncates its f32 sum: hundreds of them in one accumulator shrink it
        //      by a few parts in 10^6. So each iteration sums its own pages, small parts first, and the running
        //      totals take that sum with a rounding addition. ----
#pragma unroll
        for (int pair = 0; pair < G / 2; ++pair) {   // two groups: one 16-byte load of codes
          float cu[2][4], cr[2][4];
          uint32_t wh[PP][2][2], wl[PP][2][2];
          uint4 w[PP];
#pragma unroll
          for (int u = 0; u < PP; ++u) {
            w[u] = *reinterpret_cast<const uint4*>(tile[u] + S::TILE + (pair * 32 + lane) * 16);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t s0 = vs0[u][pair * 2 + j], s1 = vs1[u][pair * 2 + j];
              // PAIRED: a hi column has zeros for what is subtracted and for the lo part, so wl is its hi product
              wh[u][j][0] = hmul2_u32(ph[u][0] & low, s0), wh[u][j][1] = hmul2_u32(ph[u][1] & low, s1);
              wl[u][j][0] = hfma2_u32(pl[u][0] & low, s0, hfms2_u32(ph[u][0], s0, wh[u][j][0]));
              wl[u][j][1] = hfma2_u32(pl[u][1] & low, s1, hfms2_u32(ph[u][1], s1, wh[u][j][1]));
            }
          }
#pragma unroll
          for (int u = 0; u < PP; ++u) {
            const U4Word<0x6400> c00(w[u].x), c01(w[u].y), c10(w[u].z), c11(w[u].w);
            const auto add = [&](float(&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
              if (u == 0) mma_f16_zero(c, a0, a1, a2, a3, b0, b1);   // the small parts of the weights first
              else mma_f16(c, a0, a1, a2, a3, b0, b1);
            };
            add(cu[0], c00.a_u, c01.a_u, c00.b_u, c01.b_u, wl[u][0][0], wl[u][0][1]);
            add(cr[0], c00.a_n, c01.a_n, c00.b_n, c01.b_n, wl[u][0][0], wl[u][0][1]);
            add(cu[1], c10.a_u, c11.a_u, c10.b_u, c11.b_u, wl[u][1][0], wl[u][1][1]);
            add(cr[1], c10.a_n, c11.a_n, c10.b_n, c11.b_n, wl[u][1][0], wl[u][1][1]);
            if (!PAIRED) {
              mma_f16(cu[0], c00.a_u, c01.a_u, c00.b_u, c01.b_u, wh[u][0][0], wh[u][0][1]);
              mma_f16(cr[0], c00.a_n, c01.a_n, c00.b_n, c01.b_n, wh[u][0][0], wh[u][0][1]);
              mma_f16(cu[1], c10.a_u, c11.a_u, c10.b_u, c11.b_u, wh[u][1][0], wh[u][1][1]);
              mma_f16(cr[1], c10.a_n, c11.a_n, c10.b_n, c11.b_n, wh[u][1][0], wh[u][1][1]);
            }
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              add2(o_hi[pair * 2 + j][c], o_hi[pair * 2 + j][c + 1], cu[j][c], cu[j][c + 1]);
              add2(o_lo[pair * 2 + j][c], o_lo[pair * 2 + j][c + 1], cr[j][c], cr[j][c + 1]);
            }
        }
      }
      if (again) {   // the same pages for the next class of their rows
        if (special) special_at = n;
        n -= PP;
        continue;
      }
      // the warp is done with these stages: their next pages, a lane for each
      const int next = n + SLOTS;
      __syncwarp();
      if (next < count) {   // (uniform)
        if (next - batch >= 32) {
          batch += 32;
          entries = entries_next;
          entries_next = entry_of(batch + 32 + lane);
        }
        // (32 is a multiple of PP: an iteration's entries lie in one batch)
#pragma unroll
        for (int u = 0; u < PP; ++u) {
          const int32_t page = __shfl_sync(0xffffffffu, entries, next - batch + u);
          if (next + u < count && lane == 0) fetch(at + u, page);
        }
      }
      at += PP;
      if (at == SLOTS) at = 0, phase ^= 1;
    }

    // ---- hand this warp's state to the merge buffer (it aliases the ring) ----
    __syncthreads();
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, off);
      l1 += __shfl_xor_sync(0xffffffffu, l1, off);
#pragma unroll
      for (int grp = 0; grp < G; ++grp) {
        o_b[0][grp] += __shfl_xor_sync(0xffffffffu, o_b[0][grp], off);
        o_b[1][grp] += __shfl_xor_sync(0xffffffffu, o_b[1][grp], off);
      }
    }
    if (PAIRED) {
#pragma unroll
      for (int grp = 0; grp < G; ++grp)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          o_hi[grp][c] += __shfl_xor_sync(0xffffffffu, o_hi[grp][c], 2);
          o_lo[grp][c] += __shfl_xor_sync(0xffffffffu, o_lo[grp][c], 2);
        }
    }
    float* ow = o_s + warp * 8 * S::OPAD;
#pragma unroll
    for (int grp = 0; grp < G; ++grp)
#pragma unroll
      for (int c = 0; c < 4; ++c) {   // (dim g + 8 * (c / 2); head 2t + c % 2; PAIRED: rows 4 to 7 repeat rows 0 to 3, unread)
        float* to = ow + (2 * t + (c & 1)) * S::OPAD + grp * QGROUP + g + 8 * (c >> 1);
        to[0] = o_lo[grp][c] + o_b[c & 1][grp];
        to[16] = fmaf(fmaf(o_hi[grp][c], 16777216.0f, -o_lo[grp][c]), 0.0625f, o_b[c & 1][grp]);
      }
    if (g == 0) {
      ml_s[(warp * 8 + 2 * t) * 2] = m0;
      ml_s[(warp * 8 + 2 * t) * 2 + 1] = l0;
      ml_s[(warp * 8 + 2 * t + 1) * 2] = m1;
      ml_s[(warp * 8 + 2 * t + 1) * 2 + 1] = l1;
    }
  }
  __syncthreads();
  finish_block<HD, CLUSTER, PEERS, THREADS, 1, WARPS>(a, o_s, ml_s, S::OPAD, flags, seq, kvh, split, gqa, do_append, len_ptr, len, tid,
                                   splits, recv_s);
  if (PEERS) peers_finish(a, tid, flags);
}

bool attention_u4_supported(int dtype, int head_dim, int gqa) {
  return dtype == KV_U4G32 && (head_dim == 64 || head_dim == 128 || head_dim == 256) && gqa >= 1 && gqa <= 8;
}

// The instances of one head size and group of query heads, and what they need.
struct U4Instance {
  const void* kernels[3];   // plain, cluster, peers
  int blocks_per_sm, threads, smem, cluster_smem;
};
template <int HD, bool PAIRED>
static U4Instance u4_instance() {
  return {{reinterpret_cast<const void*>(attention_u4_kernel<HD, false, false, PAIRED>),
           reinterpret_cast<const void*>(attention_u4_kernel<HD, true, false, PAIRED>),
           reinterpret_cast<const void*>(attention_u4_kernel<HD, false, true, PAIRED>)},
          U4Shape<HD>::BLOCKS, U4Shape<HD>::WARPS * 32, U4Smem<HD, false>::TOTAL, U4Smem<HD, true>::TOTAL};
}
static U4Instance u4_instance(int head_dim, int gqa) {
  if (gqa <= 4) return head_dim == 64 ? u4_instance<64, true>() : head_dim == 128 ? u4_instance<128, true>() : u4_instance<256, true>();
  return head_dim == 64 ? u4_instance<64, false>() : head_dim == 128 ? u4_instance<128, false>() : u4_instance<256, false>();
}

int attention_u4_blocks_per_sm(int head_dim) { return u4_instance(head_dim, 8).blocks_per_sm; }

int attention_u4_resident_blocks(int head_dim, int gqa, bool peers) {
  const U4Instance x = u4_instance(head_dim, gqa);
  int blocks = 0;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, x.kernels[peers ? 2 : 0], x.threads, x.smem) == cudaSuccess ? blocks : 0;
}

// How many clusters of `splits` blocks the device can hold at once (0: such a launch would fail).
int attention_u4_max_clusters(int head_dim, int gqa, int splits) {
  const U4Instance x = u4_instance(head_dim, gqa);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(splits, 1, 1);
  cfg.blockDim = dim3(x.threads);
  cfg.dynamicSmemBytes = x.cluster_smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, x.kernels[1], &cfg) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return n;
}

cudaError_t attention_u4_configure() {
  for (int i = 0; i < 6; ++i) {
    const U4Instance x = u4_instance(64 << i / 2, i % 2 ? 8 : 4);
    for (int kind = 0; kind < 3; ++kind) {
      cudaError_t e = cudaFuncSetAttribute(x.kernels[kind], cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
      // clusters of more than 8 blocks (up to 16 splits merge as one cluster) are an opt-in
      if (e == cudaSuccess && kind == 1) e = cudaFuncSetAttribute(x.kernels[kind], cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return e;
    }
  }
  return cudaSuccess;
}

cudaError_t launch_attention_u4(const AttnArgs& a, int n_seq, cudaStream_t stream) {
  const U4Instance x = u4_instance(a.pool.head_dim, a.q_heads / a.pool.kv_heads);
  const bool peers = a.n_peers > 0, cluster = a.cluster_merge && !peers;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.splits, a.pool.kv_heads, n_seq);
  cfg.blockDim = dim3(x.threads);
  cfg.dynamicSmemBytes = cluster ? x.cluster_smem : x.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n_attr = 0;
  if (cluster) {
    // the splits of a (sequence, KV head) are the x extent of the grid and of the cluster
    attr[n_attr].id = cudaLaunchAttributeClusterDimension;
    attr[n_attr].val.clusterDim.x = a.splits;
    attr[n_attr].val.clusterDim.y = 1;
    attr[n_attr].val.clusterDim.z = 1;
    n_attr += 1;
  } else if (a.shared_merge == 1) {
    // blocks that wait for one another next to launches of other streams
    attr[n_attr].id = cudaLaunchAttributeCooperative;
    attr[n_attr].val.cooperative = 1;
    n_attr += 1;
  }
  if (a.pdl_wait) {
    attr[n_attr].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n_attr].val.programmaticStreamSerializationAllowed = 1;
    n_attr += 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n_attr;
  void* args[1] = {const_cast<AttnArgs*>(&a)};
  return cudaLaunchKernelExC(&cfg, x.kernels[peers ? 2 : cluster ? 1 : 0], args);
}

}  // namespace sgk
