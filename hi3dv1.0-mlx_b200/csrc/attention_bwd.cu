// Attention backward pass for sm_100a, probabilities recomputed from the forward's log-sum-exp:
//
//   P = exp(scale Q K^T - L)    dP = dO V^T    dS = P (dP - delta),  delta = rowsum(dO O)
//   dV = P^T dO                 dK = scale dS^T Q                    dQ = scale dS K
//
// One launch holds two kinds of CTA, both 128 stationary rows against a stream of row blocks:
//
//   key CTAs    K, V stay in shared memory, (Q, dO) blocks stream past:
//               S^T = K Q^T, T = V dO^T, dV += P^T dO, dK += dS^T Q     (4 products a block)
//   query CTAs  Q, dO stay, (K, V) blocks stream past:
//               S = Q K^T, T = dO V^T, dQ += dS K                       (3 products a block)
//
// so every gradient is summed in the tensor core's fp32 accumulators in one fixed order: no
// atomics, the same bits on every run, no fp32 buffer for dQ.  The price is that S and dP are
// computed twice (7 products where 5 would do).  Grouped key heads and K/V shared by the batch
// only lengthen the key CTAs' stream: the sum over the heads of a group and over the batch is
// the same accumulation.
//
// CTA (384 threads): warp 0 loads (TMA ring of NST stages) and owns the TMEM; warps 1-3 issue the
// MMAs, one each for S, T and the accumulators, so that none queues behind another's waits (a
// wait costs 80-100 cycles even when it is over); the other eight compute, each four of them half
// of a block's columns.
// TMEM: S is double-buffered, T single, then the accumulators.  P and dS (16-bit) are written
// over the S columns that the same warp has read, and are the A operands of the last products.
// S(j+2) runs when the accumulator products of j are done with its buffer, T(j+1) as soon as T(j)
// has been read, so a compute warp finds the next block ready.
//
// What bounds it.  8192 x 16 x 64 bf16: 895 us, 768 TFLOP/s of the five products that a backward
// pass cannot do without, 1075 of the seven done (66 % of the measured burst rate, and near the
// power limit: a sustained loop runs at 1.55-1.7 GHz).  Counters at 4096: tensor pipe 47 %, FMA pipe
// 49 %, MUFU 34 %, issue 51 %, DRAM 2 %: a scheduler's two compute warps take the exponentials, then
// the products' elementwise part, in step, so no pipe is busy throughout.  Measured and not kept
// (same size): 16 compute warps of half the columns 970 us; two CTAs an SM with 64-row blocks
// 950-990 (a 64-column product reads 50 cycles' worth of shared memory in 33, and S, T and the
// accumulators then form one chain); column sets with T, or S and T, of their own so that they drift
// apart 905-935; T read before the exponentials 1044; barriers asked ahead of need 920-945.
// 2049 x 16 over 4 heads of 128: 118 us, 1020 TFLOP/s of the seven products, tensor pipe 59 %.
#include <type_traits>

#include "abi.h"
#include "common.cuh"

namespace hi3d {
namespace attn_bwd {

constexpr int kRows = 128;           // stationary rows of a CTA
constexpr float kLog2e = 1.4426950408889634f;
// Of the 16 pairs of exponentials that a thread takes, those evaluated on the FMA pipe instead of
// the MUFU unit.  8192 x 16 x 64 bf16 on one box: four 910 us, five 916, six 871, seven 889, eight 912.
constexpr int kEmuPairs = 6;
// fp16 only: P is stored times 2^kPShift (P <= 1, so at most 256), which keeps probabilities
// down to 2^-22 normal numbers; dV is divided by it at the end.
constexpr int kPShift = 8;

struct Strides {
  int64_t row, head, batch;
};

struct Params {
  void *dq, *dk, *dv;
  Strides sdq, sdk, sdv;
  const int32_t *cu_q, *cu_k;
  int64_t nq, nk;
  int num_seqs, heads, kv_heads, group;
  int kv_seqs;    // key sets: num_seqs, or 1 when all sequences share one
  int q_tiles;    // row tiles of one query head: per sequence (dense) or over all (varlen)
  int kv_tiles;   // the same of one key head
  int kv_ctas, kv_first, q_first;  // key CTAs, and where each kind begins in the grid
  int kv_splits, q_splits;
  float* part_kv;  // splits > 1: [split][2][key set][kv head][kv row][D] (dK, dV) in fp32
  float* part_q;   // [split][query batch][head][query row][D]
  // per pair of query rows {-L log2e, -L log2e, -delta, -delta}, tiles of 128 rows (fp16: + kPShift)
  const float4* stat;
  // fp16: largest finite |dO| of each statistics tile, and |V| of each tile of 128 rows of a key head
  const float *max_o, *max_v;
  const float* spoiled;  // 1 for each statistics tile that has a NaN log-sum-exp, else 0
  float scale, scale2;
};

template <int D, bool KV>
struct Cfg {
  static constexpr int NCH = (D + 63) / 64;
  static constexpr int BN = D <= 64 ? 128 : 64;  // streamed rows of a block
  static constexpr int SUB = D <= 64 ? 2 : 1;
  static constexpr int HC = 32 * SUB;            // columns of a block that one compute warp takes
  static constexpr int GROUPS = BN / HC;         // column groups of a block: 4 compute warps each
  static constexpr int THREADS = 128 + GROUPS * 128;
  static constexpr int NST = 4;
  static constexpr int X_CHUNK = kRows * 128;
  static constexpr int X_BYTES = NCH * X_CHUNK;  // one stationary operand
  static constexpr int Y_CHUNK = BN * 128;
  static constexpr int Y_BYTES = NCH * Y_CHUNK;  // one streamed operand
  static constexpr int STAT_BYTES = KV ? BN * 8 : 0;
  static constexpr int STAGE = 2 * Y_BYTES;
  static constexpr int T_COL = 2 * BN;
  static constexpr int ACC_COL = 3 * BN;  // dK or dQ, then dV
  // Stationary operands that fit beside them are copied into TMEM and read from there: a 64-column
  // product with both operands in shared memory is bound by its reads (50 cycles a K step where
  // 33 would do).  With room for one it is X2.  2049 x 16 over 4 heads of 128: 119 us, without 130.
  static constexpr int X_COL = ACC_COL + (KV ? 2 : 1) * D;
  static constexpr int X_FIT = BN == 64 ? (512 - X_COL) / (D / 2) : 0;
  static constexpr bool X1_TMEM = X_FIT >= 2, X2_TMEM = X_FIT >= 1;
  static constexpr int SMEM = 2 * X_BYTES + NST * STAGE + NST * BN * 8 + 1024 /*align*/ + 256 /*barriers*/;
  static_assert(ACC_COL + (KV ? 2 : 1) * D <= 512, "TMEM budget");
  static_assert(SMEM <= 232448, "shared memory budget");
};

struct Barriers {
  uint64_t x_full;
  uint64_t x_tmem;    // the stationary operands are in TMEM
  uint64_t full[4];
  uint64_t empty[4];
  uint64_t tail;      // a ragged block, before its rows past the end are cleared
  uint64_t s_full[2];
  uint64_t t_full;
  uint64_t t_free;    // T is in the compute warps' registers
  uint64_t pd_full[2];
  uint64_t acc_done[2];
  uint64_t drained[3];  // after a time-out: an issuing warp's products are done
  uint32_t tmem_base;
  int abort;
};

// First row tile of packed sequence b when every sequence begins at a tile of its own:
// start(b + 1) - start(b) covers len(b) rows whatever the lengths, so tiles never mix
// sequences and no longest length is needed.
__device__ __forceinline__ int tile_start(const int32_t* cu, int b, int64_t rows) {
  const int64_t at = min(max((int64_t)cu[b], (int64_t)0), rows);
  return (int)(at >> 7) + b;
}

// The sequence that owns packed tile t: the last b with tile_start(b) <= t.
__device__ __forceinline__ int find_seq(const int32_t* cu, int num_seqs, int t, int64_t rows) {
  int lo = 0, hi = num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tile_start(cu, mid, rows) <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void seq_range(const int32_t* cu, int b, int64_t rows, int64_t& start, int64_t& len) {
  start = 0, len = rows;
  if (cu) {
    start = cu[b];
    len = (int64_t)cu[b + 1] - start;
    clamp_range(start, len, rows);
  }
}

// First stat tile of (sequence, head).
__device__ __forceinline__ int64_t stat_tile(const Params& p, int b, int h) {
  return p.cu_q ? (int64_t)h * p.q_tiles + tile_start(p.cu_q, b, p.nq)
                : ((int64_t)b * p.heads + h) * p.q_tiles;
}

// The blocks that stream past one CTA, in order.  Key CTAs: for each sequence that reads the
// key set, for each head of the group, the query blocks.  Query CTAs: the key blocks.
template <int BN, bool KV>
struct Stream {
  const Params& p;
  int b, b_end, g, blk, nblk;
  int head0;
  int64_t start, len;

  __device__ __forceinline__ Stream(const Params& p_, int b0, int b1, int head) : p(p_), b(b0), b_end(b1), g(0), blk(0), head0(head) {
    load();
  }
  __device__ __forceinline__ void load() {
    nblk = 0;
    for (; b < b_end; ++b) {
      seq_range(KV ? p.cu_q : p.cu_k, b, KV ? p.nq : p.nk, start, len);
      nblk = (int)((len + BN - 1) / BN);
      if (nblk > 0) return;
    }
  }
  __device__ __forceinline__ int groups() const { return KV ? p.group : 1; }
  __device__ __forceinline__ void next() {
    if (++blk < nblk) return;
    blk = 0;
    if (++g < groups()) return;
    g = 0;
    ++b;
    load();
  }
  // all blocks of the stream (from its beginning)
  __device__ __forceinline__ int64_t count() const {
    if (!(KV ? p.cu_q : p.cu_k)) return (int64_t)(b_end - b) * groups() * nblk;
    int64_t n = 0;
    for (int i = b; i < b_end; ++i) {
      int64_t s, l;
      seq_range(KV ? p.cu_q : p.cu_k, i, KV ? p.nq : p.nk, s, l);
      n += (l + BN - 1) / BN * groups();
    }
    return n;
  }
  __device__ __forceinline__ void skip(int64_t n) {
    n += (int64_t)g * nblk + blk;
    while (b < b_end) {
      const int64_t here = (int64_t)groups() * nblk;
      if (n < here) {
        g = (int)(n / nblk);
        blk = (int)(n - (int64_t)g * nblk);
        return;
      }
      n -= here;
      g = blk = 0;
      ++b;
      load();
    }
  }
  __device__ __forceinline__ int head() const { return head0 + g; }
  __device__ __forceinline__ int batch() const { return (KV ? p.cu_q : p.cu_k) ? 0 : b; }
  __device__ __forceinline__ int row() const { return (int)(start + (int64_t)blk * BN); }
  __device__ __forceinline__ int tail() const { return (int)(len % BN); }  // rows of a ragged last block
  __device__ __forceinline__ int valid() const { return (int)min((int64_t)BN, len - (int64_t)blk * BN); }
  // this block's statistics (KV)
  __device__ __forceinline__ const float4* stat() const {
    return p.stat + (stat_tile(p, b, head()) * kRows + (int64_t)blk * BN) / 2;
  }
};

// Exponent k with 2 D max|dO| max|V| 2^k < 2^15: |dS| 2^k <= |dP| + |delta| scaled stays inside
// fp16 whatever the gradient's size, and small gradients keep their bits.
__device__ __forceinline__ int ds_exponent(float max_o, float max_v, int D) {
  const float bound = 2.0f * D * max_o * max_v;
  if (!(bound > 0.0f)) return 0;
  const int k = 14 - ilogbf(fminf(bound, 1e30f));
  return min(max(k, -40), 40);
}

// The largest of runs * inner tile maxima, `outer` from run to run, by a whole warp.
__device__ __forceinline__ float fold_max(const float* m, int64_t outer, int inner, int runs) {
  float x = 0.f;
  for (unsigned e = threadIdx.x & 31; e < (unsigned)(inner * runs); e += 32)
    x = fmaxf(x, m[(int64_t)(e / (unsigned)inner) * outer + e % (unsigned)inner]);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, i));
  return x;
}
// [first, first + count) tiles of sequences [b0, b1) in one head's tiles
__device__ __forceinline__ void tile_range(const int32_t* cu, int b0, int b1, int64_t rows, int& first, int& count) {
  first = tile_start(cu, b0, rows);
  count = max(tile_start(cu, b1, rows) - first, 0);
}

// 32 lanes x 32 fp32 columns, and 32 lanes x 16 columns of packed 16-bit pairs.  BY_COLUMN: a
// thread holds four rows of eight columns (two halves of 16 lanes), else one row.
template <bool BY_COLUMN>
__device__ __forceinline__ void load_block(uint32_t taddr, uint32_t (&r)[32]) {
  if constexpr (BY_COLUMN) {
    tmem_ld_16x256b_x4(taddr, *reinterpret_cast<uint32_t(*)[16]>(&r[0]));
    tmem_ld_16x256b_x4(taddr + (16u << 16), *reinterpret_cast<uint32_t(*)[16]>(&r[16]));
  } else {
    tmem_ld32(taddr, r);
  }
}
template <bool BY_COLUMN>
__device__ __forceinline__ void store_block(uint32_t taddr, const uint32_t (&r)[16]) {
  if constexpr (BY_COLUMN) {
    tmem_st_16x128b_x4(taddr, *reinterpret_cast<const uint32_t(*)[8]>(&r[0]));
    tmem_st_16x128b_x4(taddr + (16u << 16), *reinterpret_cast<const uint32_t(*)[8]>(&r[8]));
  } else {
    tmem_st16(taddr, r);
  }
}

template <typename T, int D, bool KV>
__device__ __forceinline__ void role(const CUtensorMap* tmX1, const CUtensorMap* tmX2, const CUtensorMap* tmY1,
                                     const CUtensorMap* tmY2, const Params& p, int cta, uint8_t* smem) {
  using C = Cfg<D, KV>;
  constexpr int BN = C::BN, HC = C::HC, SUB = C::SUB, NST = C::NST, kGroups = C::GROUPS, kThreads = C::THREADS;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  uint8_t* sX1 = smem;              // K or Q
  uint8_t* sX2 = sX1 + C::X_BYTES;  // V or dO
  uint8_t* sY = sX2 + C::X_BYTES;   // [NST]{Q or K, dO or V}
  uint8_t* sStat = sY + NST * C::STAGE;
  Barriers* bar = reinterpret_cast<Barriers*>(sStat + NST * BN * 8);

  // ---- this CTA's rows
  const int splits = KV ? p.kv_splits : p.q_splits;
  const int split = cta % splits;
  cta /= splits;
  const int tiles = KV ? p.kv_tiles : p.q_tiles;
  const int32_t* cu = KV ? p.cu_k : p.cu_q;
  const int64_t rows = KV ? p.nk : p.nq;
  int t = cta % tiles;
  cta /= tiles;
  const int xheads = KV ? p.kv_heads : p.heads;
  const int h = cta % xheads;
  int seq = cta / xheads;  // sequence (query CTAs) or key set (key CTAs); varlen: 0
  if (cu) {
    seq = find_seq(cu, p.num_seqs, t, rows);
    t -= tile_start(cu, seq, rows);
  }
  int64_t x_start, x_len;
  seq_range(cu, seq, rows, x_start, x_len);
  const int64_t row0 = (int64_t)t * kRows;
  if (t < 0 || row0 >= x_len) return;  // uniform across the CTA
  const int x_batch = cu ? 0 : seq;

  // ---- what streams past it
  int b0 = seq, b1 = seq + 1;
  if (KV && p.kv_seqs == 1 && !p.cu_k) b0 = 0, b1 = p.num_seqs;           // shared keys: all sequences
  if (!KV && p.kv_seqs == 1 && !p.cu_k) b0 = 0, b1 = 1;                   // the one key set
  Stream<BN, KV> it(p, b0, b1, KV ? h * p.group : h / p.group);
  const int64_t total = it.count();
  const int64_t first = total * split / splits;
  const int n = (int)(total * (split + 1) / splits - first);
  it.skip(first);

  const int warp = warp_id(), lane = lane_id();
  const bool partial = splits > 1;
  if (n == 0) {
    // nothing to sum: zeros
    constexpr int V = D / 8;
    for (int e = threadIdx.x; e < kRows * V; e += kThreads) {
      const int64_t r = row0 + e / V;
      const int d = e % V * 8;
      if (r >= x_len) break;
#pragma unroll
      for (int w = 0; w < (KV ? 2 : 1); ++w) {
        if (partial) {
          float* part = KV ? p.part_kv : p.part_q;
          const int64_t set = (int64_t)split * (KV ? 2 : 1) + w, sets = KV ? p.kv_seqs : p.num_seqs;
          float* dst = part + (((set * (cu ? 1 : sets) + x_batch) * xheads + h) * rows + x_start + r) * D + d;
          *reinterpret_cast<float4*>(dst) = make_float4(0.f, 0.f, 0.f, 0.f);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
          const Strides& s = !KV ? p.sdq : w == 0 ? p.sdk : p.sdv;
          T* dst = static_cast<T*>(!KV ? p.dq : w == 0 ? p.dk : p.dv) + x_batch * s.batch + (x_start + r) * s.row +
                   (int64_t)h * s.head + d;
          *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
        }
      }
    }
    return;
  }

  if (threadIdx.x == 0) {
    mbar_init(&bar->x_full, 1);
    mbar_init(&bar->x_tmem, 4 * kGroups);
    for (int s = 0; s < NST; ++s) {
      mbar_init(&bar->full[s], 1);
      mbar_init(&bar->empty[s], 1);
    }
    mbar_init(&bar->tail, 1);
    for (int i = 0; i < 3; ++i) mbar_init(&bar->drained[i], 1);
    mbar_init(&bar->t_full, 1);
    mbar_init(&bar->t_free, 4 * kGroups);  // one arrival per compute warp
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->s_full[i], 1);
      mbar_init(&bar->pd_full[i], 4 * kGroups);
      mbar_init(&bar->acc_done[i], 1);
    }
    bar->abort = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(&bar->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bar->tmem_base;
  volatile int* abort = &bar->abort;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      mbar_arrive_expect_tx(&bar->x_full, 2 * C::X_BYTES);
      for (int c = 0; c < C::NCH; ++c) {
        tma_load_4d(sX1 + c * C::X_CHUNK, tmX1, &bar->x_full, c * 64, (int)(x_start + row0), h, x_batch);
        tma_load_4d(sX2 + c * C::X_CHUNK, tmX2, &bar->x_full, c * 64, (int)(x_start + row0), h, x_batch);
      }
    }
    const bool ragged = (KV ? p.cu_q : p.cu_k) != nullptr;
    int issued = 0, tails = 0;
    for (int j = 0; j < n; ++j, it.next()) {
      const int s = j % NST;
      if (!warp_wait(&bar->empty[s], ((j / NST) & 1) ^ 1, abort, 301)) break;
      uint8_t* y = sY + s * C::STAGE;
      const int valid = it.valid();
      // Rows past a packed sequence's end are the next sequence's: they are cleared, since a
      // NaN or infinity there times P = 0 would not be 0.  (Rows past the tensor are 0 anyway.)
      const bool clear = ragged && valid < BN;
      uint64_t* fb = clear ? &bar->tail : &bar->full[s];
      if (lane == 0) {
        mbar_arrive_expect_tx(fb, C::STAGE + C::STAT_BYTES);
        for (int c = 0; c < C::NCH; ++c) {
          tma_load_4d(y + c * C::Y_CHUNK, tmY1, fb, c * 64, it.row(), it.head(), it.batch());
          tma_load_4d(y + C::Y_BYTES + c * C::Y_CHUNK, tmY2, fb, c * 64, it.row(), it.head(), it.batch());
        }
        if constexpr (KV) bulk_load(sStat + s * BN * 8, it.stat(), C::STAT_BYTES, fb);
      }
      if (clear) {
        volatile int no_abort = 0;
        warp_wait(&bar->tail, tails & 1, &no_abort, 302);
        ++tails;
        for (int c = 0; c < 2 * C::NCH; ++c)
          for (int e = valid * 8 + lane; e < BN * 8; e += 32)
            *reinterpret_cast<uint4*>(y + c * C::Y_CHUNK + e * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->full[s]);
      }
      issued = j + 1;
    }
    if (__any_sync(0xffffffffu, *abort)) {
      // let every copy already issued land before the CTA exits
      volatile int no_abort = 0;
      warp_wait(&bar->x_full, 0, &no_abort, 303);
      for (int j = issued > NST ? issued - NST : 0; j < issued; ++j)
        warp_wait(&bar->full[j % NST], (j / NST) & 1, &no_abort, 304);
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------ MMA issuers
    const int role_id = warp - 1;
    // The whole warp runs the loop and one elected lane issues: under `if (lane == 0)` the compiler
    // does not know that descriptors and addresses are the same in all active lanes, and an MMA
    // costs 50 cycles and more to issue (measured alone, 64 columns: 53 cycles against 33).
    {
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t idesc_s = make_idesc(1, fmt, 0, 0, kRows, BN);
      constexpr uint32_t idesc_acc = make_idesc(1, fmt, 0, 1, kRows, D);
      const uint64_t dX1 = smem_desc(smem_u32(sX1), 16, 1024, kLayoutSW128);
      const uint64_t dX2 = smem_desc(smem_u32(sX2), 16, 1024, kLayoutSW128);
      const uint64_t dY = smem_desc(smem_u32(sY), 16, 1024, kLayoutSW128);
      const uint64_t dYt = smem_desc(smem_u32(sY), C::Y_CHUNK, 1024, kLayoutSW128);  // rows as the K dimension
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      // d = x y^T over the channels, x in TMEM (x_col) or in shared memory
      auto product = [&](auto in_tmem, uint32_t d, uint64_t x, uint32_t x_col, uint32_t y_off,
                         uint64_t* done) {
        if (!elect_one()) return;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint64_t y = dY + ((y_off + (ks >> 2) * C::Y_CHUNK + (ks & 3) * 32) >> 4);
          if constexpr (decltype(in_tmem)::value)
            mma_f16_ts(d, x_col + ks * 8, y, idesc_s, ks > 0 ? 1u : 0u);
          else
            mma_f16_ss(d, x + (((ks >> 2) * C::X_CHUNK + (ks & 3) * 32) >> 4), y, idesc_s, ks > 0 ? 1u : 0u);
        }
        tc_commit(done);
      };
      using X1InTmem = std::integral_constant<bool, C::X1_TMEM>;
      using X2InTmem = std::integral_constant<bool, C::X2_TMEM>;
      const uint32_t x2_col = tm + C::X_COL, x1_col = x2_col + D / 2;
      // acc += a y over the block's rows; a: HC / 2 TMEM columns in each group of the S buffer
      auto accumulate = [&](uint32_t d, uint32_t a, uint32_t y_off, bool more) {
#pragma unroll
        for (int ks = 0; ks < BN / 16; ++ks) {
          const int group = ks / (HC / 16), k = ks % (HC / 16);
          mma_f16_ts(d, a + group * HC + k * 8, dYt + ((y_off + ks * 2048) >> 4), idesc_acc, more || ks > 0 ? 1u : 0u);
        }
      };
      if (role_id != 2) mbar_wait(C::X2_TMEM ? &bar->x_tmem : &bar->x_full, 0, abort, 310);
      if (C::X2_TMEM && !C::X1_TMEM && role_id == 0) mbar_wait(&bar->x_full, 0, abort, 310);
      for (int j = 0; j < n; ++j) {
        const uint32_t y = (j % NST) * C::STAGE;
        mbar_wait(&bar->full[j % NST], (j / NST) & 1, abort, 311);
        if (role_id == 0) {  // S(j), once the products that read P(j - 2), dS(j - 2) from this buffer are done
          if (j > 1) mbar_wait(&bar->acc_done[j & 1], ((j - 2) >> 1) & 1, abort, 314);
          tc_fence_after();
          product(X1InTmem(), tm + (j & 1) * BN, dX1, x1_col, y, &bar->s_full[j & 1]);
        } else if (role_id == 1) {  // T(j), once T(j - 1) has been read
          if (j > 0) mbar_wait(&bar->t_free, (j - 1) & 1, abort, 312);
          tc_fence_after();
          product(X2InTmem(), tm + C::T_COL, dX2, x2_col, y + C::Y_BYTES, &bar->t_full);
        } else {  // the accumulators, once P(j), dS(j) are written
          mbar_wait(&bar->pd_full[j & 1], (j >> 1) & 1, abort, 313);
          tc_fence_after();
          const uint32_t a = tm + (j & 1) * BN;
          if (elect_one()) {
            accumulate(tm + C::ACC_COL, a + HC / 2, y, j > 0);
            if constexpr (KV) accumulate(tm + C::ACC_COL + D, a, y + C::Y_BYTES, j > 0);
            tc_commit(&bar->acc_done[j & 1]);
            if (j + NST < n) tc_commit(&bar->empty[j % NST]);
          }
        }
        __syncwarp();
      }
      if (__any_sync(0xffffffffu, *abort)) {
        // products were issued on whatever their buffers held: they end before the CTA's memory goes
        volatile int no_abort = 0;
        if (elect_one()) tc_commit(&bar->drained[role_id]);
        warp_wait(&bar->drained[role_id], 0, &no_abort, 315);
      }
    }
  } else {
    // ------------------------------------------------------------ compute
    const int group = (warp - 4) >> 2;
    const int sub = warp & 3;
    const int row = sub * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(sub * 32) << 16;
    const uint32_t tT = tmem + lane_addr + C::T_COL + group * HC;
    const uint64_t scale2x2 = f2_splat(p.scale2);
    // The exponent that dS carries, from the rows that enter this CTA's sums alone: another sequence's,
    // head's or (query CTAs) row tile's sizes do not cost these their bits.
    int kexp = 0;
    // the largest of a value of each statistics tile that this CTA's sums run over
    auto over_tiles = [&](const float* m) {
      int first = 0, count = p.q_tiles;
      if constexpr (!KV) return m[stat_tile(p, seq, h) + t];
      if (p.cu_q) {
        tile_range(p.cu_q, b0, b1, p.nq, first, count);
        return fold_max(m + (int64_t)h * p.group * p.q_tiles + first, p.q_tiles, count, p.group);
      }
      return fold_max(m + ((int64_t)b0 * p.heads + h * p.group) * p.q_tiles, (int64_t)p.heads * p.q_tiles,
                      p.group * p.q_tiles, b1 - b0);
    };
    if constexpr (kHalf) {
      const int hk = KV ? h : h / p.group, set = p.kv_seqs == 1 ? 0 : seq;
      int vt = 0, nv = p.kv_tiles;
      if (p.cu_k) tile_range(p.cu_k, seq, seq + 1, p.nk, vt, nv);
      const float max_v = fold_max(p.max_v + ((int64_t)(p.cu_k ? 0 : set) * p.kv_heads + hk) * p.kv_tiles + vt, 0, nv, 1);
      kexp = ds_exponent(over_tiles(p.max_o), max_v, D);
    }
    // A NaN log-sum-exp must reach dV through every P of its row, also those that the polynomial would
    // make finite (dK and dQ have it from delta): such CTAs take the exponentials of the masked form.
    const bool spoiled = KV && over_tiles(p.spoiled) > 0.f;
    // key CTAs keep P 2^kPShift in 16 bits: dS takes the rest of its exponent here
    const uint64_t gain = f2_splat(ldexpf(1.0f, kexp - kPShift));
    // query CTAs: this row's statistics, the exponent of dS inside the probability's
    float nl = -INFINITY, nd = 0.f;
    if (!KV && row0 + row < x_len) {
      const float4 st = p.stat[(stat_tile(p, seq, h) * kRows + row0 + row) / 2];
      nl = ((row & 1) ? st.y : st.x) + (kHalf ? (float)(kexp - kPShift) : 0.f);
      nd = (row & 1) ? st.w : st.z;
    }
    const uint64_t nl2 = f2_splat(nl), nd2 = f2_splat(nd);
    // A thread holds 16 pairs of neighbouring columns, pair e in registers 2 e, 2 e + 1.  Query CTAs
    // (statistics by row): one row, columns 2 e, 2 e + 1.  Key CTAs (statistics by column): four
    // rows of eight columns, column 8 k + 2 (lane % 4) with k = (e / 2) % 4, so that four 16-byte
    // shared loads serve a block where one row a thread needs 32 (which bound the kernel: a
    // broadcast still moves 16 bytes to each lane).
    const int col0 = KV ? 2 * (lane & 3) : 0;
    auto column = [&](int e) { return col0 + (KV ? 8 * ((e >> 1) & 3) : 2 * e); };
    // One block; MASK: only its first `valid` rows are the sequence's, all exponentials by the MUFU unit.
    auto block = [&](int j, int valid, auto mask) {
      constexpr bool MASK = decltype(mask)::value;
      const uint32_t tS = tmem + lane_addr + (j & 1) * BN + group * HC;
      const float4* st = reinterpret_cast<const float4*>(sStat + (j % NST) * BN * 8) + group * (HC / 2) + (lane & 3);
      float4 q[4];
      uint32_t sv[SUB][32], pk[16];
      if (KV) mbar_wait(&bar->full[j % NST], (j / NST) & 1, abort, 320);
      mbar_wait(&bar->s_full[j & 1], (j >> 1) & 1, abort, 321);
      tc_fence_after();
#pragma unroll
      for (int u = 0; u < SUB; ++u) load_block<KV>(tS + u * 32, sv[u]);
      tmem_wait_ld();
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        if constexpr (KV) {
#pragma unroll
          for (int k = 0; k < 4; ++k) q[k] = st[u * 16 + 4 * k];
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          uint64_t bias = nl2;
          if constexpr (KV) bias = f2_pack(q[(e >> 1) & 3].x, q[(e >> 1) & 3].y);
          const uint64_t x =
              f2_fma(f2_pack(__uint_as_float(sv[u][2 * e]), __uint_as_float(sv[u][2 * e + 1])), scale2x2, bias);
          float p0, p1;
          if (!MASK && e * kEmuPairs % 16 < kEmuPairs) {  // spread over the 16
            f2_unpack(f2_exp2_poly(x), p0, p1);
          } else {
            f2_unpack(x, p0, p1);
            p0 = ex2_approx(p0), p1 = ex2_approx(p1);
          }
          if constexpr (MASK) {  // past the end: not a probability, whatever the scores were
            const int c = u * 32 + column(e) + group * HC;
            p0 = c < valid ? p0 : 0.f;
            p1 = c + 1 < valid ? p1 : 0.f;
          }
          sv[u][2 * e] = __float_as_uint(p0);
          sv[u][2 * e + 1] = __float_as_uint(p1);
          if constexpr (KV) pk[e] = Cvt<T>::pack2(p0, p1);
        }
        if constexpr (KV) store_block<KV>(tS + u * 16, pk);
      }
      mbar_wait(&bar->t_full, j & 1, abort, 322);
      tc_fence_after();
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        uint32_t tv[32];
        load_block<KV>(tT + u * 32, tv);
        if constexpr (KV && SUB > 1) {
#pragma unroll
          for (int k = 0; k < 4; ++k) q[k] = st[u * 16 + 4 * k];
        }
        tmem_wait_ld();
        if (u == SUB - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->t_free);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          uint64_t d = nd2;
          if constexpr (KV) d = f2_pack(q[(e >> 1) & 3].z, q[(e >> 1) & 3].w);
          uint64_t pr = f2_pack(__uint_as_float(sv[u][2 * e]), __uint_as_float(sv[u][2 * e + 1]));
          if constexpr (KV && kHalf) pr = f2_mul(pr, gain);
          pk[e] = Cvt<T>::from_f2(
              f2_mul(pr, f2_add(f2_pack(__uint_as_float(tv[2 * e]), __uint_as_float(tv[2 * e + 1])), d)));
          if constexpr (MASK) {
            const int c = u * 32 + column(e) + group * HC;
            if (c >= valid) pk[e] &= 0xffff0000u;
            if (c + 1 >= valid) pk[e] &= 0x0000ffffu;
          }
        }
        store_block<KV>(tS + HC / 2 + u * 16, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar->pd_full[j & 1]);
    };
    if constexpr (C::X2_TMEM) {
      // this warp's rows of the stationary operands, the column groups one chunk of 64 channels each
      if (warp_wait(&bar->x_full, 0, abort, 324)) {
#pragma unroll
        for (int x = 0; x < (C::X1_TMEM ? 2 : 1); ++x)
          for (int c = group; c < C::NCH; c += kGroups) {
            const uint8_t* src = (x == 0 ? sX2 : sX1) + c * C::X_CHUNK + row * 128;
            const uint32_t dst = tmem + lane_addr + C::X_COL + x * (D / 2) + c * 32;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (c * 64 + half * 32 >= D) break;
              uint32_t v[16];
#pragma unroll
              for (int k = 0; k < 4; ++k)  // 128-byte swizzle: 16-byte unit u of row r lies at u ^ (r % 8)
                *reinterpret_cast<uint4*>(&v[4 * k]) =
                    *reinterpret_cast<const uint4*>(src + (((half * 4 + k) ^ (row & 7)) << 4));
              tmem_st16(dst + half * 16, v);
            }
          }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->x_tmem);
      }
    }
    for (int j = 0; j < n;) {
      // the blocks of one sequence and head; its last may be ragged
      const int m = min(n - j, it.nblk - it.blk), whole = (int)(it.len / BN) - it.blk;
      for (int i = 0; i < m; ++i, ++j) {
        if (i < whole && !spoiled)
          block(j, BN, std::false_type());
        else
          block(j, i < whole ? BN : it.tail(), std::true_type());
      }
      it.skip(m);
    }
    // ---- epilogue: the groups alternate, W channels at a time
    if (!__any_sync(0xffffffffu, *abort) && warp_wait(&bar->acc_done[(n - 1) & 1], ((n - 1) >> 1) & 1, abort, 323)) {
      tc_fence_after();
      const int64_t r = row0 + row;
      const float mul = p.scale * ldexpf(1.0f, -kexp);
#pragma unroll
      for (int w = 0; w < (KV ? 2 : 1); ++w) {
        const float f = w == 0 ? mul : kHalf ? ldexpf(1.0f, -kPShift) : 1.0f;
        const Strides& s = !KV ? p.sdq : w == 0 ? p.sdk : p.sdv;
        T* dst = static_cast<T*>(!KV ? p.dq : w == 0 ? p.dk : p.dv) + x_batch * s.batch + (x_start + r) * s.row +
                 (int64_t)h * s.head;
        float* part = KV ? p.part_kv : p.part_q;
        const int64_t set = (int64_t)split * (KV ? 2 : 1) + w, sets = KV ? p.kv_seqs : p.num_seqs;
        part += (((set * (cu ? 1 : sets) + x_batch) * xheads + h) * rows + x_start + r) * D;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          constexpr int W = 32 / kGroups;
          static_assert(W == 16, "one 16-column load a group");
          const int d0 = c * 32 + group * W;
          uint32_t v[W];
          __syncwarp();
          tmem_ld16(tmem + lane_addr + C::ACC_COL + w * D + d0, v);
          tmem_wait_ld();
          if (r < x_len) {
            if (partial) {
#pragma unroll
              for (int e = 0; e < W; e += 4)
                *reinterpret_cast<float4*>(part + d0 + e) =
                    make_float4(__uint_as_float(v[e]) * f, __uint_as_float(v[e + 1]) * f,
                                __uint_as_float(v[e + 2]) * f, __uint_as_float(v[e + 3]) * f);
            } else {
#pragma unroll
              for (int e = 0; e < W; e += 8) {
                uint4 o;
                o.x = Cvt<T>::pack2(__uint_as_float(v[e]) * f, __uint_as_float(v[e + 1]) * f);
                o.y = Cvt<T>::pack2(__uint_as_float(v[e + 2]) * f, __uint_as_float(v[e + 3]) * f);
                o.z = Cvt<T>::pack2(__uint_as_float(v[e + 4]) * f, __uint_as_float(v[e + 5]) * f);
                o.w = Cvt<T>::pack2(__uint_as_float(v[e + 6]) * f, __uint_as_float(v[e + 7]) * f);
                *reinterpret_cast<uint4*>(dst + d0 + e) = o;
              }
            }
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D, true>::THREADS, 1)
    bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO,
               const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
               const __grid_constant__ CUtensorMap tmQs, const __grid_constant__ CUtensorMap tmDOs,
               const __grid_constant__ CUtensorMap tmKs, const __grid_constant__ CUtensorMap tmVs,
               const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int keys = (int)blockIdx.x - p.kv_first;
  if (keys >= 0 && keys < p.kv_ctas)
    role<T, D, true>(&tmK, &tmV, &tmQs, &tmDOs, p, keys, smem);
  else
    role<T, D, false>(&tmQ, &tmDO, &tmKs, &tmVs, p, blockIdx.x - p.q_first, smem);
}

// Over this many keys or fewer delta is summed from P and dP (below).
constexpr int kFewKeys = 16;
// CTAs an SM: the kernel is short and waits for its loads.  8192 x 16 x 64 bf16: eight 8.4 us (32
// registers, a little spilled), six 11.4, unbounded 15.3.  The form for few keys needs registers:
// 16384 x 16 queries on 16 keys, the whole pass, four 200 us, five 202, six 211; packed 5873 x 22 x 96
// fp16, this kernel, 23.2, 21.8, 21.0 (23.6 with five since it also takes its tiles' maxima).
constexpr int kStatCtas = 8, kFewCtas = 5;

// Row statistics {-L log2e, -delta} in tiles of 128 rows, delta = rowsum(dO O) in fp32.  Over few
// keys delta nearly cancels dP, and O's rounding in it would be most of dS's error (dQ in bf16, 512
// queries: 2 keys 0.0040 relative, 5 0.0029, 16 and more 0.0025): there delta = sum P dP / sum P,
// the products done again here, 16 FMAs a key and 8 channels (then 0.0024 throughout; 4096 x 16 queries,
// the whole pass: 4 keys 45 us, 16 keys 62, 36 without).  Blocks
// [0, stat_blocks): one (tile, head, sequence) each; rows past the sequence's end get
// probability 0.  fp16: these blocks also take their tile's largest finite |dO|, and the blocks after
// them the largest finite |V| of each tile of a key head (tiles as the key CTAs').
// Reads O and dO once: 4096 x 16 x 64 bf16 7.2 us, 8192 8.4 us (4.0 TB/s; short, so its launch, the
// first loads' latency and the tail count as much as the bytes).
struct StatParams {
  const void *o, *d_o, *q, *k, *v;
  Strides so, sdo, sq, sk, sv;
  const float* lse;
  float* stat;
  float *max_o, *max_v, *spoiled;
  int stat_blocks;
};

template <typename T, int D>
__device__ __forceinline__ float abs_max8(uint4 u, float m) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f2_unpack(Cvt<T>::to_f2(w[i]), a, b);
    a = fabsf(a), b = fabsf(b);
    if (a < INFINITY) m = fmaxf(m, a);
    if (b < INFINITY) m = fmaxf(m, b);
  }
  return m;
}

// Products of 8 channels, summed
template <typename T>
__device__ __forceinline__ float dot8(uint4 a, uint4 b) {
  uint64_t sum = f2_mul(Cvt<T>::to_f2(a.x), Cvt<T>::to_f2(b.x));
  sum = f2_fma(Cvt<T>::to_f2(a.y), Cvt<T>::to_f2(b.y), sum);
  sum = f2_fma(Cvt<T>::to_f2(a.z), Cvt<T>::to_f2(b.z), sum);
  sum = f2_fma(Cvt<T>::to_f2(a.w), Cvt<T>::to_f2(b.w), sum);
  float x, y;
  f2_unpack(sum, x, y);
  return x + y;
}

// One value pair of a tile's row
__device__ __forceinline__ void put_stat(const StatParams& q, int64_t tile, int r, float l, float delta) {
  float* dst = q.stat + (tile * kRows + (r & ~1)) * 2 + (r & 1);
  dst[0] = l, dst[2] = delta;
}

// The statistics of a tile whose sequence has at most kFewKeys keys.  Four keys at a time: their
// eight products are summed across a row's lanes by a transposing exchange (8 shuffles where a sum
// each would take 24), after which a lane has one key.
template <typename T, int D>
__device__ __forceinline__ void few_keys(const Params& p, const StatParams& q, int t, int h, int b, int64_t tile,
                                         float& big, bool& nan) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr int L = D == 64 ? 8 : 16;
  constexpr float shift = kHalf ? (float)kPShift : 0.f;
  constexpr uint32_t kAll = 0xffffffffu;
  const int sub = threadIdx.x % L, batch = p.cu_q ? 0 : b, kb = p.cu_k || p.kv_seqs == 1 ? 0 : b;
  const bool dp_lane = sub & 4, high2 = sub & 2, high1 = sub & 1;
  int64_t start, len, k_start, keys;
  seq_range(p.cu_q, b, p.nq, start, len);
  seq_range(p.cu_k, b, p.nk, k_start, keys);
  const T* x = static_cast<const T*>(q.q) + batch * q.sq.batch + (int64_t)h * q.sq.head + sub * 8;
  const T* d = static_cast<const T*>(q.d_o) + batch * q.sdo.batch + (int64_t)h * q.sdo.head + sub * 8;
  const T* k = static_cast<const T*>(q.k) + kb * q.sk.batch + (int64_t)(h / p.group) * q.sk.head + sub * 8;
  const T* v = static_cast<const T*>(q.v) + kb * q.sv.batch + (int64_t)(h / p.group) * q.sv.head + sub * 8;
#pragma unroll 1
  for (int r = threadIdx.x / L; r < kRows; r += 256 / L) {
    const int64_t row = (int64_t)t * kRows + r;
    const bool in = row < len && sub * 8 < D;
    float sum = 0.f, delta = 0.f, l = 0.f;
    if (__any_sync(kAll, in)) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      const uint4 a = in ? *reinterpret_cast<const uint4*>(x + (start + row) * q.sq.row) : zero;
      const uint4 g = in ? *reinterpret_cast<const uint4*>(d + (start + row) * q.sdo.row) : zero;
      if (row < len) l = q.lse[((int64_t)batch * p.heads + h) * p.nq + start + row] * kLog2e;
      nan = nan || l != l;
      if constexpr (kHalf) big = abs_max8<T, D>(g, big);
#pragma unroll 1
      for (int j = 0; j < (int)keys; j += 4) {
        float e8[8], e4[4], e2[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool have = in && j + i < (int)keys;
          e8[i] = dot8<T>(a, have ? *reinterpret_cast<const uint4*>(k + (k_start + j + i) * q.sk.row) : zero);
          e8[i + 4] = dot8<T>(g, have ? *reinterpret_cast<const uint4*>(v + (k_start + j + i) * q.sv.row) : zero);
        }
        if constexpr (L == 16) {
#pragma unroll
          for (int i = 0; i < 8; ++i) e8[i] += __shfl_xor_sync(kAll, e8[i], 8);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          e4[i] = (dp_lane ? e8[i + 4] : e8[i]) + __shfl_xor_sync(kAll, dp_lane ? e8[i] : e8[i + 4], 4);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          e2[i] = (high2 ? e4[i + 2] : e4[i]) + __shfl_xor_sync(kAll, high2 ? e4[i] : e4[i + 2], 2);
        const float mine = (high1 ? e2[1] : e2[0]) + __shfl_xor_sync(kAll, high1 ? e2[0] : e2[1], 1);
        const float other = __shfl_xor_sync(kAll, mine, 4);
        const float pr =
            j + (sub & 3) < (int)keys ? exp2f(fmaf(dp_lane ? other : mine, p.scale2, -l)) : 0.f;
        sum += pr, delta = fmaf(pr, dp_lane ? mine : other, delta);
      }
#pragma unroll
      for (int m = 2; m > 0; m >>= 1) {
        sum += __shfl_xor_sync(kAll, sum, m);
        delta += __shfl_xor_sync(kAll, delta, m);
      }
    }
    // sum is 1 up to the log-sum-exp's rounding, which must not part delta from dP
    if (sub == 0) put_stat(q, tile, r, row < len ? shift - l : -INFINITY, row < len && keys > 0 ? -delta / sum : 0.f);
  }
}

// FEW: some sequence may have that few keys.
template <typename T, int D, bool FEW>
__global__ void __launch_bounds__(256, FEW ? kFewCtas : kStatCtas)
    stat_kernel(const __grid_constant__ Params p, const __grid_constant__ StatParams q) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr int L = D == 64 ? 8 : 16;  // lanes of a row, 8 channels each (96: 12 of 16 work)
  const int sub = threadIdx.x % L;
  const bool on = sub * 8 < D;
  constexpr float shift = kHalf ? (float)kPShift : 0.f;  // the exponent that P carries in 16 bits
  float big = 0.f;
  bool nan = false;
  if ((int)blockIdx.x < q.stat_blocks) {
    int t = blockIdx.x % p.q_tiles, rest = blockIdx.x / p.q_tiles;
    const int64_t tile = blockIdx.x;
    const int h = rest % p.heads;
    int b = rest / p.heads;
    if (p.cu_q) {
      b = find_seq(p.cu_q, p.num_seqs, t, p.nq);
      t -= tile_start(p.cu_q, b, p.nq);
    }
    int64_t start, len;
    seq_range(p.cu_q, b, p.nq, start, len);
    const int batch = p.cu_q ? 0 : b;
    if (t < 0 || (int64_t)t * kRows >= len) {
      if (threadIdx.x == 0) {
        q.spoiled[tile] = 0.f;
        if (kHalf) q.max_o[tile] = 0.f;
      }
      return;
    }
    const T* o = static_cast<const T*>(q.o) + batch * q.so.batch + (int64_t)h * q.so.head + sub * 8;
    const T* d = static_cast<const T*>(q.d_o) + batch * q.sdo.batch + (int64_t)h * q.sdo.head + sub * 8;
    int64_t k_start, keys = p.nk;
    if (FEW) seq_range(p.cu_k, b, p.nk, k_start, keys);
    if (FEW && keys <= kFewKeys) {
      few_keys<T, D>(p, q, t, h, b, tile, big, nan);
    } else {
#pragma unroll 4
      for (int r = threadIdx.x / L; r < kRows; r += 256 / L) {
        const int64_t row = (int64_t)t * kRows + r;
        float acc = 0.f;
        if (row < len && on) {
          const uint4 a = *reinterpret_cast<const uint4*>(o + (start + row) * q.so.row);
          const uint4 g = *reinterpret_cast<const uint4*>(d + (start + row) * q.sdo.row);
          acc = dot8<T>(a, g);
          if constexpr (kHalf) big = abs_max8<T, D>(g, big);
        }
#pragma unroll
        for (int m = L / 2; m > 0; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
        if (sub == 0) {
          const float l = row < len ? q.lse[((int64_t)batch * p.heads + h) * p.nq + start + row] : INFINITY;
          nan = nan || l != l;
          put_stat(q, tile, r, shift - l * kLog2e, row < len ? -acc : 0.f);
        }
      }
    }
    const int any = __syncthreads_or(nan);
    if (threadIdx.x == 0) q.spoiled[tile] = any ? 1.f : 0.f;
  } else {
    const int blk = blockIdx.x - q.stat_blocks;
    int t = blk % p.kv_tiles;
    const int h = blk / p.kv_tiles % p.kv_heads, b = blk / p.kv_tiles / p.kv_heads;
    int64_t start = 0, len = p.nk;
    if (p.cu_k) {
      const int seq = find_seq(p.cu_k, p.num_seqs, t, p.nk);
      t -= tile_start(p.cu_k, seq, p.nk);
      seq_range(p.cu_k, seq, p.nk, start, len);
    }
    const T* v = static_cast<const T*>(q.v) + (int64_t)b * q.sv.batch + (int64_t)h * q.sv.head + sub * 8;
    for (int r = threadIdx.x / L; t >= 0 && r < kRows; r += 256 / L) {
      const int64_t row = (int64_t)t * kRows + r;
      if (row < len && on) big = abs_max8<T, D>(*reinterpret_cast<const uint4*>(v + (start + row) * q.sv.row), big);
    }
  }
  if constexpr (kHalf) {
    __shared__ float most[8];
    for (int m = 16; m > 0; m >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, m));
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = big;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < 8; ++w) big = fmaxf(big, most[w]);
      if ((int)blockIdx.x < q.stat_blocks)
        q.max_o[blockIdx.x] = big;
      else
        q.max_v[blockIdx.x - q.stat_blocks] = big;
    }
  }
}

// Sums the fp32 partials of the splits in order and rounds them: out[batch][row][head][D].  8 bytes
// of partials a split and value of dK, dV: two splits of 2049 x 4 x 128, 5.5 us.  Rows before the first
// packed sequence and after the last have no partials and are left alone.
struct ReduceJob {
  const float* part;
  void* out;
  Strides s;
  int64_t rows;
  int heads, batches, splits;
  int64_t split_stride;  // floats between two splits
  int64_t items;         // batches * heads * rows * D / 8
  const int32_t* cu;     // packed rows: [num_seqs + 1] offsets
  int num_seqs;
};

template <typename T, int D>
__global__ void __launch_bounds__(256) reduce_kernel(const ReduceJob j0, const ReduceJob j1, const ReduceJob j2) {
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const ReduceJob* j = &j0;
  if (i >= j->items) i -= j->items, j = &j1;
  if (j == &j1 && i >= j->items) i -= j->items, j = &j2;
  if (i >= j->items) return;
  const int d = (int)(i % (D / 8)) * 8;
  int64_t rest = i / (D / 8);
  const int64_t row = rest % j->rows;
  rest /= j->rows;
  if (j->cu && (row < j->cu[0] || row >= j->cu[j->num_seqs])) return;
  const float* src = j->part + i * 8;
  float a[8] = {};
  for (int s = 0; s < j->splits; ++s, src += j->split_stride) {
    const float4 x = *reinterpret_cast<const float4*>(src), y = *reinterpret_cast<const float4*>(src + 4);
    a[0] += x.x, a[1] += x.y, a[2] += x.z, a[3] += x.w, a[4] += y.x, a[5] += y.y, a[6] += y.z, a[7] += y.w;
  }
  T* dst = static_cast<T*>(j->out) + rest / j->heads * j->s.batch + row * j->s.row + rest % j->heads * j->s.head + d;
  uint4 o;
  o.x = Cvt<T>::pack2(a[0], a[1]);
  o.y = Cvt<T>::pack2(a[2], a[3]);
  o.z = Cvt<T>::pack2(a[4], a[5]);
  o.w = Cvt<T>::pack2(a[6], a[7]);
  *reinterpret_cast<uint4*>(dst) = o;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct Plan {
  int q_tiles, kv_tiles, kv_seqs, q_batches, kv_batches;
  int64_t kv_ctas, q_ctas;
  // The kind with the longer streams starts first, so that none begins late.  64 queries on 8192
  // keys, 16 heads of 64, bf16: 58 us, with the key CTAs first 101.
  bool q_first;
  int kv_splits, q_splits;
  int64_t max_o, max_v;                 // fp16: tile maxima
  int64_t max_bytes, stat_bytes;
  int64_t kv_part, q_part;              // floats of one split's partials
  int64_t bytes;
};

static int64_t round256(int64_t b) { return (b + 255) & ~int64_t(255); }

// How many CTAs share one tile's stream.  A CTA should not take longer than the mean load of an
// SM (`ideal`, in blocks): a short key set under many queries (cross-attention), or a handful of
// tiles, would otherwise leave most SMs idle behind a few long streams.  Each split costs a write
// and a read of fp32 partials and one more launch, so a stream may be kSlack longer, and a part
// keeps at least kMinBlocks blocks.  Whole backward pass in bf16, split against never split: 8192
// queries on 77 keys, 16 heads of 64, 61 us against 77; 4 heads 26 against 72; 2049 x 8 over one key
// head of 64 50 against 149; 2049 x 16 over 4 heads of 64 (kept whole) 81, split 86.
static int split_count(int64_t steps, double ideal) {
  constexpr int kMinBlocks = 4;
  constexpr double kSlack = 1.1;
  if (steps <= kSlack * ideal || steps < 2 * kMinBlocks) return 1;
  const int64_t want = (int64_t)(steps / (ideal > kMinBlocks ? ideal : kMinBlocks) + 0.999);
  return (int)(want < 1 ? 1 : want > 64 ? 64 : want);
}

static Plan make_plan(const hi3d_attn_bwd_args* a) {
  Plan n;
  const bool vq = a->cu_seqlens_q != nullptr, vk = a->cu_seqlens_k != nullptr;
  const bool shared = !vk && (a->k_batch == 0 || a->num_seqs == 1);
  n.kv_seqs = shared ? 1 : a->num_seqs;
  n.q_tiles = (int)(vq ? (a->nq >> 7) + a->num_seqs : (a->nq + 127) / 128);
  n.kv_tiles = (int)(vk ? (a->nk >> 7) + a->num_seqs : (a->nk + 127) / 128);
  n.q_batches = vq ? 1 : a->num_seqs;
  n.kv_batches = vk ? 1 : n.kv_seqs;
  const int bn = a->head_dim <= 64 ? 128 : 64;
  // blocks of one CTA's stream (packed sequences: their mean, the lengths are on the device)
  const int64_t group = a->heads / a->kv_heads;
  const int64_t q_blocks = (a->nq + bn - 1) / bn, k_blocks = (a->nk + bn - 1) / bn;
  const int64_t kv_steps = group * (vq ? (shared ? q_blocks + a->num_seqs : (q_blocks + a->num_seqs - 1) / a->num_seqs)
                                       : q_blocks * (shared ? a->num_seqs : 1));
  const int64_t q_steps = vk ? (k_blocks + a->num_seqs - 1) / a->num_seqs : k_blocks;
  const int64_t kv_tiles = (int64_t)n.kv_tiles * a->kv_heads * n.kv_batches;
  const int64_t q_tiles = (int64_t)n.q_tiles * a->heads * n.q_batches;
  constexpr double kQueryCost = 0.8;       // a query block has 3 products where a key block has 4
  const double setup = bn == 128 ? 6 : 8;  // a CTA's set-up and epilogue, about 7 us
  const double load = kv_tiles * (kv_steps + setup) + q_tiles * (kQueryCost * q_steps + setup);
  const double ideal = load / sm_count();
  n.kv_splits = split_count(kv_steps, ideal);
  n.q_splits = split_count(q_steps, ideal / kQueryCost);
  n.kv_ctas = kv_tiles * n.kv_splits;
  n.q_ctas = q_tiles * n.q_splits;
  n.q_first = kQueryCost * q_steps / n.q_splits > (double)kv_steps / n.kv_splits;
  const int64_t stat_tiles = (int64_t)n.q_tiles * a->heads * n.q_batches;
  const bool half = a->dtype == HI3D_F16;
  n.max_o = half ? stat_tiles : 0, n.max_v = half ? kv_tiles : 0;
  n.max_bytes = round256((n.max_o + n.max_v + stat_tiles) * 4);
  n.stat_bytes = round256(stat_tiles * kRows * 8);
  n.kv_part = (int64_t)n.kv_batches * a->kv_heads * a->nk * a->head_dim;
  n.q_part = (int64_t)n.q_batches * a->heads * a->nq * a->head_dim;
  n.bytes = n.max_bytes + n.stat_bytes + (n.kv_splits > 1 ? round256(n.kv_part * 2 * n.kv_splits * 4) : 0) +
            (n.q_splits > 1 ? round256(n.q_part * n.q_splits * 4) : 0);
  return n;
}

static int check_args(const hi3d_attn_bwd_args* a) {
  if (!a || !a->q || !a->k || !a->v || !a->out || !a->dout || !a->lse || !a->dq || !a->dk || !a->dv)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: null pointer");
  if (a->dtype != HI3D_F16 && a->dtype != HI3D_BF16)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: dtype must be f16 or bf16");
  if (a->head_dim != 64 && a->head_dim != 96 && a->head_dim != 128)
    return set_error(HI3D_ERR_UNSUPPORTED, "flash_attn_bwd: head_dim %d not supported (64, 96, 128)", a->head_dim);
  if (a->num_seqs < 1 || a->heads < 1 || a->nq < 1 || a->nk < 1)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: sizes must be positive");
  if (a->kv_heads < 1 || a->heads % a->kv_heads)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: %d key heads do not divide %d query heads",
                     a->kv_heads, a->heads);
  const void* ptrs[] = {a->q, a->k, a->v, a->out, a->dout, a->dq, a->dk, a->dv};
  for (const void* x : ptrs)
    if (!aligned16(x)) return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: pointers must be 16-byte aligned");
  const int64_t strides[] = {a->q_row,  a->q_head,  a->q_batch,  a->k_row,  a->k_head,  a->k_batch,
                             a->v_row,  a->v_head,  a->v_batch,  a->o_row,  a->o_head,  a->o_batch,
                             a->do_row, a->do_head, a->do_batch, a->dq_row, a->dq_head, a->dq_batch,
                             a->dk_row, a->dk_head, a->dk_batch, a->dv_row, a->dv_head, a->dv_batch};
  for (int64_t s : strides)
    if (s < 0 || s % 8) return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: strides must be multiples of 8");
  if (!(a->scale >= 0.f) || a->scale > 3.0e38f)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: scale must be finite and not negative");
  if (!a->cu_seqlens_q && a->cu_seqlens_k)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: packed keys need packed queries");
  if (a->nq > 0x7ffffff0 || a->nk > 0x7ffffff0)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: more than 2^31 rows");
  return HI3D_OK;
}

template <typename T, int D>
static int launch(const hi3d_attn_bwd_args* a, const Plan& n, uint8_t* ws, cudaStream_t st) {
  using CK = Cfg<D, true>;
  const int64_t qb = n.q_batches, kb = n.kv_batches;
  constexpr int BN = CK::BN;
  CUtensorMap mq, md, mk, mv, mqs, mds, mks, mvs;
  int rc;
  if ((rc = make_attn_map(&mq, a->q, a->dtype, D, a->nq, a->heads, qb, a->q_row, a->q_head, a->q_batch, kRows)) ||
      (rc = make_attn_map(&md, a->dout, a->dtype, D, a->nq, a->heads, qb, a->do_row, a->do_head, a->do_batch,
                          kRows)) ||
      (rc = make_attn_map(&mk, a->k, a->dtype, D, a->nk, a->kv_heads, kb, a->k_row, a->k_head, a->k_batch, kRows)) ||
      (rc = make_attn_map(&mv, a->v, a->dtype, D, a->nk, a->kv_heads, kb, a->v_row, a->v_head, a->v_batch, kRows)))
    return rc;
  if (BN == kRows) {
    mqs = mq, mds = md, mks = mk, mvs = mv;
  } else if ((rc = make_attn_map(&mqs, a->q, a->dtype, D, a->nq, a->heads, qb, a->q_row, a->q_head, a->q_batch, BN)) ||
             (rc = make_attn_map(&mds, a->dout, a->dtype, D, a->nq, a->heads, qb, a->do_row, a->do_head, a->do_batch,
                                 BN)) ||
             (rc = make_attn_map(&mks, a->k, a->dtype, D, a->nk, a->kv_heads, kb, a->k_row, a->k_head, a->k_batch,
                                 BN)) ||
             (rc = make_attn_map(&mvs, a->v, a->dtype, D, a->nk, a->kv_heads, kb, a->v_row, a->v_head, a->v_batch,
                                 BN))) {
    return rc;
  }
  Params p;
  p.dq = a->dq, p.dk = a->dk, p.dv = a->dv;
  p.sdq = {a->dq_row, a->dq_head, a->dq_batch};
  p.sdk = {a->dk_row, a->dk_head, a->dk_batch};
  p.sdv = {a->dv_row, a->dv_head, a->dv_batch};
  p.cu_q = a->cu_seqlens_q, p.cu_k = a->cu_seqlens_k;
  p.nq = a->nq, p.nk = a->nk;
  p.num_seqs = a->num_seqs, p.heads = a->heads, p.kv_heads = a->kv_heads, p.group = a->heads / a->kv_heads;
  p.kv_seqs = n.kv_seqs;
  p.q_tiles = n.q_tiles, p.kv_tiles = n.kv_tiles;
  p.kv_ctas = (int)n.kv_ctas, p.kv_first = n.q_first ? (int)n.q_ctas : 0, p.q_first = n.q_first ? 0 : (int)n.kv_ctas;
  p.kv_splits = n.kv_splits, p.q_splits = n.q_splits;
  p.scale = a->scale, p.scale2 = a->scale * kLog2e;
  float* const max_o = reinterpret_cast<float*>(ws);
  p.max_o = max_o, p.max_v = max_o + n.max_o, p.spoiled = max_o + n.max_o + n.max_v;
  p.stat = reinterpret_cast<const float4*>(ws + n.max_bytes);
  p.part_kv = reinterpret_cast<float*>(ws + n.max_bytes + n.stat_bytes);
  p.part_q = p.part_kv + (n.kv_splits > 1 ? round256(n.kv_part * 2 * n.kv_splits * 4) / 4 : 0);

  StatParams q;
  q.o = a->out, q.d_o = a->dout, q.q = a->q, q.k = a->k, q.v = a->v;
  q.so = {a->o_row, a->o_head, a->o_batch};
  q.sdo = {a->do_row, a->do_head, a->do_batch};
  q.sq = {a->q_row, a->q_head, a->q_batch};
  q.sk = {a->k_row, a->k_head, a->k_batch};
  q.sv = {a->v_row, a->v_head, a->v_batch};
  q.lse = a->lse;
  q.stat = reinterpret_cast<float*>(ws + n.max_bytes);
  q.max_o = max_o, q.max_v = max_o + n.max_o, q.spoiled = max_o + n.max_o + n.max_v;
  q.stat_blocks = (int)((int64_t)n.q_tiles * a->heads * qb);
  const int64_t blocks = q.stat_blocks + n.max_v;
  if (a->cu_seqlens_k || a->nk <= kFewKeys)
    stat_kernel<T, D, true><<<(unsigned)blocks, 256, 0, st>>>(p, q);
  else
    stat_kernel<T, D, false><<<(unsigned)blocks, 256, 0, st>>>(p, q);
  if ((rc = check_launch("flash_attn_bwd statistics"))) return rc;

  auto kern = bwd_kernel<T, D>;
  static bool allowed[64];
  if ((rc = allow_shared(reinterpret_cast<const void*>(kern), CK::SMEM, allowed, "flash_attn_bwd"))) return rc;
  kern<<<(unsigned)(n.kv_ctas + n.q_ctas), CK::THREADS, CK::SMEM, st>>>(mq, md, mk, mv, mqs, mds, mks, mvs, p);
  if ((rc = check_launch("flash_attn_bwd"))) return rc;

  ReduceJob jobs[3] = {};
  if (n.kv_splits > 1)
    for (int w = 0; w < 2; ++w)
      jobs[w] = {p.part_kv + w * n.kv_part, w == 0 ? a->dk : a->dv, w == 0 ? p.sdk : p.sdv, a->nk, a->kv_heads,
                 n.kv_batches, n.kv_splits, 2 * n.kv_part, n.kv_part / 8, a->cu_seqlens_k, a->num_seqs};
  if (n.q_splits > 1)
    jobs[2] = {p.part_q,   a->dq,    p.sdq,           a->nq,          a->heads,   n.q_batches,
               n.q_splits, n.q_part, n.q_part / 8, a->cu_seqlens_q, a->num_seqs};
  const int64_t items = jobs[0].items + jobs[1].items + jobs[2].items;
  if (items == 0) return HI3D_OK;
  reduce_kernel<T, D><<<(unsigned)((items + 255) / 256), 256, 0, st>>>(jobs[0], jobs[1], jobs[2]);
  return check_launch("flash_attn_bwd reduction");
}

template <typename T>
static int dispatch(const hi3d_attn_bwd_args* a, const Plan& n, uint8_t* ws, cudaStream_t st) {
  switch (a->head_dim) {
    case 64: return launch<T, 64>(a, n, ws, st);
    case 96: return launch<T, 96>(a, n, ws, st);
    default: return launch<T, 128>(a, n, ws, st);
  }
}

}  // namespace attn_bwd
}  // namespace hi3d

using namespace hi3d;

extern "C" int hi3d_flash_attn_bwd_workspace_size(const hi3d_attn_bwd_args* a, int64_t* bytes) {
  int rc = attn_bwd::check_args(a);
  if (rc) return rc;
  if (!bytes) return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: null bytes");
  *bytes = attn_bwd::make_plan(a).bytes;
  return HI3D_OK;
}

extern "C" int hi3d_flash_attn_bwd(const hi3d_attn_bwd_args* a, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  int rc = attn_bwd::check_args(a);
  if (rc) return rc;
  const attn_bwd::Plan n = attn_bwd::make_plan(a);
  if (n.kv_ctas + n.q_ctas > 0x7fffffff)
    return set_error(HI3D_ERR_INVALID_ARGUMENT, "flash_attn_bwd: too many tiles");
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || workspace_bytes < n.bytes)
    return set_error(HI3D_ERR_CAPACITY, "flash_attn_bwd: workspace %lld bytes, need %lld (256-byte aligned)",
                     (long long)workspace_bytes, (long long)n.bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t st = as_stream(stream);
  return a->dtype == HI3D_BF16 ? attn_bwd::dispatch<__nv_bfloat16>(a, n, ws, st)
                               : attn_bwd::dispatch<__half>(a, n, ws, st);
}
