// Attention of many query rows over packed sequences or a paged cache
// (cmpx_attention_seq) on the tensor cores: fp16 / bf16, head_dim 64 or 128.
// No counterpart in the reference.
//
//   O_i = sum_j softmax_j(scale * Q_i . K_j) V_j over the keys row i sees
//
// Rows.  The query heads of one kv head share its keys, so a tile's 128 rows
// are (token, head of the group) pairs: floor(128 / group) tokens, every head
// of the group.  A chunk of few tokens fills as many rows as it can, and the
// causal edge of a tile spans few keys.  A thread block owns two such tiles
// (A and B, consecutive tokens of one sequence and kv head) and walks the key
// blocks of 128 that any of its rows sees.
//
// Per key block and tile the tensor core computes S = Q K^T (512 cycles at
// D = 128) and O += P V (512), and 128 threads, one a row, turn S into P:
// 16384 exponentials at 16 a cycle are 1024 cycles.  Two tiles in turn keep
// both units busy.  Measured: 4300 cycles a key block of both tiles (2048
// would be the units' own time), 566-583 us and 910-937 TFLOP/s on two prompts
// of 8192 tokens, 16 / 4 heads of 128, at clocks that the power limit holds
// near 1.6 GHz; what is left is each tile's chain of softmax (1800 cycles),
// P V, its completion and the next Q K^T (1500).  S is read into registers and
// P written over it in tensor memory, from where the P V product takes it as
// its A operand: P crosses neither shared memory, whose bandwidth the two
// products' operands need (the same product from shared memory would read 64 KB
// a block and tile instead of 32), nor a proxy fence.
//
// Running maximum: O is rescaled only when a row's maximum grew by more than
// 2^8 over the one its weights are taken against (fp32 sums and 16-bit
// weights up to 2^8 lose nothing by it; the final division by the sum of the
// same weights makes the result independent of the reference point).  A block
// after the first ones rarely does, so the read-modify-write of O in tensor
// memory leaves the loop.
//
// Warps: 0 loads (TMA; a page of the cache is one box) and clears the value
// rows behind the last visible key of the last block (what the cache or the
// next sequence holds there may be NaN, and 0 * NaN is NaN), 1 issues the
// products, 2 and 3 clear output rows that no sequence holds, 4-7 and 8-11
// softmax and output of tiles A and B; with an 8-bit cache 12-15 turn e4m3
// codes and their scales into the queries' type in shared memory (exact: a
// power of two times four significant bits).
//
// Values that are not finite and that some rows of a tile see and others do
// not (a causal edge) still reach every row through 0 * NaN.  Finite inputs
// never pay for that: a row whose result is not finite although its sum is,
// and that has such a value among the keys it may not see, is computed again
// from its definition, one warp a row.
//
// Few tiles: the key blocks of a tile are split among gridDim.z thread
// blocks, which write unnormalised sums, maxima and fp32 accumulators to the
// workspace; attention_seq_combine joins them in a fixed order.
#include <cuda_fp8.h>

#include <type_traits>

#include "attention_math.cuh"
#include "attention_seq.h"
#include "ptx.cuh"

namespace cmpx {
namespace {

template <int D, bool Q8>
struct TileCfg {
  static constexpr int WARPS = Q8 ? 16 : 12;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int QCH = D / 64;            // 128-byte chunks of a 16-bit row
  static constexpr int TILE = 128 * D * 2;      // 128 rows
  // key and value blocks in the queries' type; 8-bit codes arrive in RS raw
  // blocks, keys and values in turn (two of them left the SM waiting for one
  // load at a time, which took longer than a block's products; a key block is
  // done with early, so one converted one is enough)
  static constexpr int KS = D == 64 ? 4 : Q8 ? 1 : 3;
  static constexpr int VS = D == 64 ? 4 : 2;
  static constexpr int RS = !Q8 ? 0 : D == 64 ? 8 : 4;
  static constexpr int RAW = 128 * D;
  static constexpr size_t SMEM = size_t(TILE) * (2 + KS + VS) + size_t(RS) * (RAW + 128) + 1024 + 512;
  // registers a thread of the two softmax warpgroups and of the others
  // (setmaxnreg), out of the block's 3 x 168 or 4 x 128 at launch
  static constexpr int REGS_SOFTMAX = Q8 ? 184 : 216, REGS_OTHER = 72;
  static constexpr int REGS_NEED = 2 * REGS_SOFTMAX + (WARPS / 4 - 2) * REGS_OTHER;
  static_assert(SMEM <= 232448, "shared memory budget");
};

struct TileParams {
  SeqProblem p;
  int tokens;      // query tokens of a tile: floor(128 / group)
  int box_rows;    // keys of one TMA box (a page, or a whole block)
  int splits;
  float* part_o;   // [splits][tokens_q * heads_q][D]
  float2* part_ml; // [splits][tokens_q * heads_q]: maximum (log2 units), sum
  int* err;
};

// A warpgroup's registers a thread, given up to or taken from the block's own.
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// Zeros in the rows that no sequence holds, heads of kv head hk: this block's
// share of them over the grid's x axis, by `threads` threads.  A padded batch
// has far more such rows than others, and blocks without a tile then: those
// clear with all their threads, the others with two warps that have nothing
// else to do (at a block's end, by all its warps, it cost 8 x 1024 tokens
// without padding 1.5%).  16384 tokens of 32 heads of 128, 300 of them in a
// sequence: 0.09 ms, of which clearing 0.03; 3.4 ms by one block a kv head.
template <typename T, int D>
__device__ __forceinline__ void clear_rest(const SeqProblem& p, int hk, int thread, int threads) {
  const int2 rest = seq_rest(p);
  const int before = min(rest.x, rest.y < rest.x ? p.tokens_q : rest.x);
  const int from = rest.y < rest.x ? p.tokens_q : rest.y;
  const int outside = rest.y < rest.x ? p.tokens_q : before + (p.tokens_q - from);
  const int units = p.group * (D / 8);  // of 8 values, of one token (8 at least)
  const int step = min(units, threads), tokens = threads / step;
  const int u0 = thread % step, t0 = thread / step;
  const bool wide = (p.o_token | p.o_head) % 8 == 0 && reinterpret_cast<uintptr_t>(p.O) % 16 == 0;
  if (t0 >= tokens) return;
  // (every gridDim.x-th of them, however many threads this block has for it)
  for (int64_t o = blockIdx.x + int64_t(gridDim.x) * t0; o < outside; o += int64_t(gridDim.x) * tokens) {
    const int64_t tok = rest.y < rest.x || o < before ? o : from + (o - before);
    T* row = static_cast<T*>(p.O) + tok * p.o_token + int64_t(hk * p.group) * p.o_head;
    for (int u = u0; u < units; u += step) {
      T* at = row + (u / (D / 8)) * p.o_head + u % (D / 8) * 8;
      if (wide) {
        *reinterpret_cast<uint4*>(at) = make_uint4(0u, 0u, 0u, 0u);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) stf(at + i, 0.0f);
      }
    }
  }
}

template <int FMT, int D, bool Q8>
__global__ void __launch_bounds__(TileCfg<D, Q8>::THREADS, 1)
    attention_tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                          const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TileParams a) {
  using Cfg = TileCfg<D, Q8>;
  using T = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
  constexpr int KS = Cfg::KS, VS = Cfg::VS, RS = Cfg::RS > 0 ? Cfg::RS : 1;
  constexpr uint32_t IDESC_QK = make_idesc(uint32_t(FMT), 0u, 0u, 128, 128);
  constexpr uint32_t IDESC_PV = make_idesc(uint32_t(FMT), 0u, 1u, 128, D);
  const SeqProblem& p = a.p;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024 - (raw_addr & 1023)) & 1023);
  uint8_t* sQ = smem;                       // [2] tiles
  uint8_t* sK = sQ + 2 * Cfg::TILE;         // [KS]
  uint8_t* sV = sK + KS * Cfg::TILE;        // [VS]
  uint8_t* sR = sV + VS * Cfg::TILE;        // [RS] raw codes
  uint8_t* sScale = sR + Cfg::RS * Cfg::RAW;  // [RS][128] their e8m0 bytes
  uint64_t* bars = reinterpret_cast<uint64_t*>(sScale + Cfg::RS * 128);
  uint64_t* q_full = bars;
  uint64_t* k_full = q_full + 1;    // [KS]
  uint64_t* k_empty = k_full + KS;  // [KS]
  uint64_t* v_full = k_empty + KS;  // [VS]
  uint64_t* v_empty = v_full + VS;  // [VS]
  uint64_t* r_full = v_empty + VS;  // [RS]
  uint64_t* r_empty = r_full + RS;  // [RS]
  uint64_t* s_full = r_empty + RS;  // [2] S of tile t is in tensor memory
  uint64_t* p_full = s_full + 2;    // [2] P of tile t is, and O is rescaled
  uint64_t* o_done = p_full + 2;    // [2] P V of tile t is accumulated
  uint64_t* tail = o_done + 2;      // value rows behind the last key are cleared
  uint64_t* drain = tail + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int* found = reinterpret_cast<int*>(tmem_holder + 2);  // [2]
  int* warp_sum = found + 2;                             // [WARPS]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < KS; ++i) {
      mbar_init(&k_full[i], Q8 ? 128 : 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < VS; ++i) {
      mbar_init(&v_full[i], Q8 ? 128 : 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < RS; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], 128);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 128);
      mbar_init(&o_done[t], 1);
    }
    mbar_init(tail, 32);
    mbar_init(drain, 1);
    *abort_flag = 0;
    found[0] = -1;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_holder, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  pdl_trigger();
  pdl_wait();

  // ---- which tiles: the grid's x axis counts token tiles over all sequences,
  // late ones (which see more keys) first
  const int per_cta = 2 * a.tokens;
  const int idx = int(gridDim.x - 1 - blockIdx.x);
  for (int base = 0, total = 0; base < p.batch; base += Cfg::THREADS) {
    const int b = base + int(threadIdx.x);
    int c = 0;
    if (b < p.batch) c = (seq_queries(p, b).y + per_cta - 1) / per_cta;
    int inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    int before = total, all = total;
#pragma unroll
    for (int w = 0; w < Cfg::WARPS; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    const int rel = idx - (before + inc - c);
    if (rel >= 0 && rel < c) {
      found[0] = b;
      found[1] = rel;
    }
    __syncthreads();
    if (idx < all) break;
    total = all;
  }
  const int seq = found[0], hk = int(blockIdx.y);
  Seq s = {};
  int i0 = 0;       // first token of the block
  int kmax = 0;     // keys any row of it sees
  int nblk[2] = {0, 0};
  if (seq >= 0) {
    s = seq_of(p, seq);
    i0 = found[1] * per_cta;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int first = i0 + t * a.tokens;
      if (first < s.n) {
        const int lim = seq_limit(p, s, min(first + a.tokens, s.n) - 1);
        nblk[t] = (lim + 127) >> 7;
        kmax = max(kmax, lim);
      }
    }
  }
  // this block's share of the key blocks
  const int all_blocks = (kmax + 127) >> 7;
  const int share = (all_blocks + a.splits - 1) / a.splits;
  const int jb = min(int(blockIdx.z) * share, all_blocks), je = min(jb + share, all_blocks);
  const int nkv = je - jb;
  const int n0 = min(max(nblk[0] - jb, 0), nkv), n1 = min(max(nblk[1] - jb, 0), nkv);
  const int kend = min(kmax, je * 128);             // keys this block reads: [jb * 128, kend)
  const int last_keys = kend - (jb + nkv - 1) * 128;  // of the last key block (nkv > 0)

  const bool clears = p.zero_rest && a.splits == 1;  // with splits the combining kernel does
  if (clears && seq < 0) clear_rest<T, D>(p, hk, int(threadIdx.x), Cfg::THREADS);

  if (warp < 4) {
    regs_dec<Cfg::REGS_OTHER>();
  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (nkv > 0) {
      if (lane == 0) {
        prefetch_tmap(&tmQ);
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
        const int tiles = n1 > 0 ? 2 : 1;
        mbar_arrive_expect_tx(q_full, uint32_t(tiles * a.tokens * p.group * D * 2));
        for (int t = 0; t < tiles; ++t)
#pragma unroll
          for (int c = 0; c < Cfg::QCH; ++c)
            tma_load_4d(sQ + t * Cfg::TILE + c * 16384, &tmQ, q_full, c * 64, 0, hk, s.q0 + i0 + t * a.tokens);
      }
      // lane i loads box i of a block: page i of its pages, or the whole block
      const int boxes_full = 128 / a.box_rows;
      const int* table = p.table != nullptr ? p.table + seq * p.table_stride : nullptr;
      auto page_of = [&](int j) -> int {
        const int key = (jb + j) * 128 + lane * a.box_rows;
        if (table == nullptr || lane >= boxes_full || key >= kend) return 0;
        return __ldg(table + (key >> p.page_lg));
      };
      int page = page_of(0), kdone = 0, vdone = 0;
      bool ok = true;
      for (int j = 0; j < nkv && ok; ++j) {
        const int kv0 = (jb + j) * 128;
        const int boxes = min(boxes_full, (kend - kv0 + a.box_rows - 1) / a.box_rows);
        const int next = j + 1 < nkv ? page_of(j + 1) : 0;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          uint64_t *full, *empty;
          uint8_t* dst;
          int use;
          if constexpr (Q8) {
            const int r = (2 * j + v) % RS;
            full = &r_full[r];
            empty = &r_empty[r];
            dst = sR + r * Cfg::RAW;
            use = (2 * j + v) / RS;
          } else if (v == 0) {
            full = &k_full[j % KS];
            empty = &k_empty[j % KS];
            dst = sK + (j % KS) * Cfg::TILE;
            use = j / KS;
          } else {
            full = &v_full[j % VS];
            empty = &v_empty[j % VS];
            dst = sV + (j % VS) * Cfg::TILE;
            use = j / VS;
          }
          if (!__all_sync(0xffffffffu, mbar_wait(empty, (use & 1) ^ 1, abort_flag))) {
            if (lane == 0) rec_err(a.err, abort_flag, kDevTimeoutEmpty);
            ok = false;
            break;
          }
          // scales of pages that are none: zeros, as TMA gives for their codes
          const bool there = lane < boxes && page >= 0 && page < p.pages;
          uint32_t bytes = uint32_t(boxes * a.box_rows * D * (Q8 ? 1 : 2));
          uint8_t* sdst = sScale + ((2 * j + v) % RS) * 128 + lane * a.box_rows;
          if constexpr (Q8) {
            if (lane < boxes && !there) {
              for (int k = 0; k < a.box_rows; k += 4) *reinterpret_cast<uint32_t*>(sdst + k) = 0u;
              fence_proxy_async_smem();  // before a later copy writes the place
            }
            bytes += uint32_t(__popc(__ballot_sync(0xffffffffu, there)) * a.box_rows);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(full, bytes);
          __syncwarp();
          if (lane < boxes) {
            const CUtensorMap* m = v ? &tmV : &tmK;
            const int row = table != nullptr ? (kv0 + lane * a.box_rows) & (p.page_size - 1) : s.k0 + kv0;
            if constexpr (Q8) {
              const SeqKV& kv = v ? p.v : p.k;
              tma_load_4d(dst + lane * a.box_rows * D, m, full, 0, row, hk, page);
              if (there)
                bulk_load(sdst, kv.scale + page * kv.s_page + hk * kv.s_head + row, uint32_t(a.box_rows), full);
            } else {
#pragma unroll
              for (int c = 0; c < Cfg::QCH; ++c)
                tma_load_4d(dst + c * 16384 + lane * a.box_rows * 128, m, full, c * 64, row, hk, page);
            }
          }
          if (v == 0) ++kdone; else ++vdone;
        }
        page = next;
      }
      if (!Q8 && ok && last_keys < 128) {
        // value rows behind the last key, up to where the product stops
        const int j = nkv - 1;
        if (__all_sync(0xffffffffu, mbar_wait(&v_full[j % VS], (j / VS) & 1, abort_flag))) {
          uint8_t* v = sV + (j % VS) * Cfg::TILE;
          const int rows = ((last_keys + 15) & ~15) - last_keys;
          for (int i = lane; i < rows * 8 * Cfg::QCH; i += 32)
            *reinterpret_cast<uint4*>(v + (i / (rows * 8)) * 16384 + last_keys * 128 + (i % (rows * 8)) * 16) =
                make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          mbar_arrive(tail);
        } else if (lane == 0) {
          rec_err(a.err, abort_flag, kDevTimeoutFull);
        }
      }
      if (!ok && lane == 0) {
        // let the copies in flight land before the block exits (bounded waits;
        // a slot's loads complete in order, so the last of each is enough)
        volatile int never = 0;
        mbar_wait(q_full, 0, &never);
        if constexpr (Q8) {
          const int n = kdone + vdone;
          for (int i = n > RS ? n - RS : 0; i < n; ++i) mbar_wait(&r_full[i % RS], (i / RS) & 1, &never);
        } else {
          for (int i = kdone > KS ? kdone - KS : 0; i < kdone; ++i) mbar_wait(&k_full[i % KS], (i / KS) & 1, &never);
          for (int i = vdone > VS ? vdone - VS : 0; i < vdone; ++i) mbar_wait(&v_full[i % VS], (i / VS) & 1, &never);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ products
    // the whole warp walks along, one lane issues
    if (nkv > 0) {
      const uint32_t one = elect_one();
      auto ready = [&](uint64_t* bar, int phase) -> bool {
        return __all_sync(0xffffffffu, mbar_test_wait(bar, uint32_t(phase & 1)));
      };
      auto wait = [&](uint64_t* bar, int phase) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(bar, uint32_t(phase & 1), abort_flag));
      };
      bool ok = wait(q_full, 0);
      if (!ok) rec_err(a.err, abort_flag, kDevTimeoutFull);
      const int n[2] = {n0, n1};
      int qk[2] = {0, 0}, pv[2] = {0, 0};  // products issued
      int k_rel = 0, v_rel = 0;            // key / value blocks released
      // S = Q K^T of tile t's next block, if its keys are there.  The tile's
      // last P V must be done: P lies where S goes.
      auto issue_qk = [&](int t) -> bool {
        const int j = qk[t];
        if (!ready(&k_full[j % KS], j / KS)) return false;
        tc_fence_after();
        const uint32_t q_addr = smem_u32(sQ + t * Cfg::TILE);
        const uint32_t k_addr = smem_u32(sK + (j % KS) * Cfg::TILE);
#pragma unroll
        for (int c = 0; c < Cfg::QCH; ++c)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f16_one(one, tmem_base + uint32_t(t * 128), make_sdesc_sw128(q_addr + c * 16384 + kk * 32, 16, 1024),
                    make_sdesc_sw128(k_addr + c * 16384 + kk * 32, 16, 1024), IDESC_QK, (c | kk) != 0 ? 1u : 0u);
        mma_commit_one(one, &s_full[t]);
        ++qk[t];
        while (k_rel < nkv && (qk[0] > k_rel || n0 <= k_rel) && (qk[1] > k_rel || n1 <= k_rel)) {
          mma_commit_one(one, &k_empty[k_rel % KS]);
          ++k_rel;
        }
        return true;
      };
      // A tile's P V and next Q K^T go out together, so that the two tiles
      // fall out of step: one is in softmax while the other's products run
      // (issued as they became ready, both tiles' softmax ran at once and the
      // tensor core waited: 5500 cycles a block of both, now 4300).
      uint32_t idle = 0;  // polls since the last product
      uint64_t t0 = 0;
      while (ok && (pv[0] < n0 || pv[1] < n1)) {
        bool any = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (qk[t] == pv[t]) {
            if (qk[t] < n[t]) any = issue_qk(t) || any;
            continue;
          }
          const int j = pv[t];
          const bool cleared = Q8 || j + 1 < nkv || last_keys == 128 || ready(tail, 0);
          if (!cleared || !ready(&p_full[t], j) || !ready(&v_full[j % VS], j / VS)) continue;
          tc_fence_after();
          const uint32_t v_addr = smem_u32(sV + (j % VS) * Cfg::TILE);
          const int steps = j + 1 < nkv ? 8 : (last_keys + 15) >> 4;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            if (kk < steps)
              mma_f16_ts_one(one, tmem_base + 256u + uint32_t(t * D), tmem_base + uint32_t(t * 128 + kk * 8),
                         make_sdesc_sw128(v_addr + kk * 2048, 16384, 1024), IDESC_PV, (j | kk) != 0 ? 1u : 0u);
          mma_commit_one(one, &o_done[t]);
          ++pv[t];
          any = true;
          while (v_rel < nkv && (pv[0] > v_rel || n0 <= v_rel) && (pv[1] > v_rel || n1 <= v_rel)) {
            mma_commit_one(one, &v_empty[v_rel % VS]);
            ++v_rel;
          }
          if (qk[t] < n[t]) {
            if (!wait(&o_done[t], j)) {
              rec_err(a.err, abort_flag, kDevTimeoutFull);
              ok = false;
              break;
            }
            issue_qk(t);
          }
        }
        idle = any ? 0 : idle + 1;
        if ((idle & 1023u) == 1023u) {
          if (idle == 1023u) t0 = globaltimer_ns();
          else if (__any_sync(0xffffffffu, *abort_flag || globaltimer_ns() - t0 > CMPX_WAIT_TIMEOUT_NS)) {
            rec_err(a.err, abort_flag, kDevTimeoutFull);
            ok = false;
          }
        }
      }
      // the last commits reach their barriers before the block may exit
      if (ok && !wait(&v_empty[(nkv - 1) % VS], (nkv - 1) / VS)) {
        rec_err(a.err, abort_flag, kDevTimeoutFull);
        ok = false;
      }
      if (!ok) {
        mma_commit_one(one, drain);
        volatile int never = 0;
        mbar_wait(drain, 0, &never);
      }
    }
  } else if (clears && seq >= 0) {
    clear_rest<T, D>(p, hk, int(threadIdx.x) - 64, 64);
  }
  } else if (warp >= 12) {
    // ------------------------------------------------------------ 8-bit codes to T
    // Eight lanes a row, 16 codes each (D = 64: four lanes); a row's two
    // halves of a 16-byte pair go out in the order that keeps the eight lanes
    // on different banks.
    if constexpr (Q8) {
      regs_dec<Cfg::REGS_OTHER>();
      constexpr int LPR = D / 16, RPI = 128 / LPR;  // lanes a row, rows a pass of the 128 threads
      const int tid = int(threadIdx.x) - 384;
      const int c16 = tid % LPR, r_in = tid / LPR;
      bool ok = true;
      for (int i = 0; i < 2 * nkv && ok; ++i) {
        const int j = i >> 1, kv0 = (jb + j) * 128;
        const bool isv = (i & 1) != 0;
        const int r = i % RS, slot = isv ? j % VS : j % KS, use = isv ? j / VS : j / KS;
        ok = __all_sync(0xffffffffu, mbar_wait(&r_full[r], (i / RS) & 1, abort_flag) &&
                                         mbar_wait(isv ? &v_empty[slot] : &k_empty[slot], (use & 1) ^ 1, abort_flag));
        if (!ok) {
          if (lane == 0) rec_err(a.err, abort_flag, kDevTimeoutFull);
          break;
        }
        const uint8_t* src = sR + r * Cfg::RAW;
        uint8_t* dst = (isv ? sV : sK) + slot * Cfg::TILE;
        // four rows' loads before their stores, which the compiler must take
        // to overlap them (one row at a time: 2400 cycles for a block's keys
        // or values, more than its products take)
        constexpr int BATCH = 4;
#pragma unroll 1
        for (int k0 = 0; k0 < 128 / RPI; k0 += BATCH) {
          uint4 codes[BATCH];
          uint32_t byte[BATCH];
          bool takes = true;
#pragma unroll
          for (int b = 0; b < BATCH; ++b) {
            const int row = (k0 + b) * RPI + r_in;
            codes[b] = *reinterpret_cast<const uint4*>(src + row * D + c16 * 16);
            byte[b] = sScale[r * 128 + row];
          }
#pragma unroll
          for (int b = 0; b < BATCH; ++b) {
            // a row behind the last key may hold anything, NaN too: zeros
            if (kv0 + (k0 + b) * RPI + r_in >= kend) {
              codes[b] = make_uint4(0u, 0u, 0u, 0u);
              byte[b] = 127;
            }
            takes = takes && scale4_takes(byte[b], (T*)nullptr);
          }
          takes = __all_sync(0xffffffffu, takes);
#pragma unroll
          for (int b = 0; b < BATCH; ++b) {
            const int row = (k0 + b) * RPI + r_in;
            const uint32_t w[4] = {codes[b].x, codes[b].y, codes[b].z, codes[b].w};
            uint32_t h[8];
            if (takes) {
#pragma unroll
              for (int e = 0; e < 4; ++e) scale4(w[e], byte[b], h[2 * e], h[2 * e + 1], (T*)nullptr);
            } else {
              const float up = e8m0_to_float(byte[b]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                h[2 * e] = dequant2(w[e] & 0xffffu, up, (T*)nullptr);
                h[2 * e + 1] = dequant2(w[e] >> 16, up, (T*)nullptr);
              }
            }
            const int unit = (c16 & 3) * 2, flip = c16 >> 2;
            uint8_t* at = dst + (c16 >> 2) * 16384 + row * 128;
            const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
            *reinterpret_cast<uint4*>(at + (((unit + flip) ^ (row & 7)) << 4)) = flip ? hi : lo;
            *reinterpret_cast<uint4*>(at + (((unit + 1 - flip) ^ (row & 7)) << 4)) = flip ? lo : hi;
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(isv ? &v_full[slot] : &k_full[slot]);
        mbar_arrive(&r_empty[r]);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax and output, one thread a row
    regs_inc<Cfg::REGS_SOFTMAX>();
    const int t = (warp - 4) >> 2, qw = warp & 3, r = qw * 32 + lane;
    const int nt = t ? n1 : n0;
    const uint32_t t_lane = tmem_base + (uint32_t(qw * 32) << 16);
    const uint32_t s_col = uint32_t(t * 128), o_col = 256u + uint32_t(t * D);
    const int token = i0 + t * a.tokens + r / p.group;  // of the sequence
    const int head = hk * p.group + r % p.group;
    const bool valid = seq >= 0 && r < a.tokens * p.group && token < s.n;
    // (rows of nothing see all keys, so that they never make a warp mask)
    const int lim = valid ? seq_limit(p, s, token) : kend;
    const float sl = p.scale_log2;
    float m = -INFINITY, l = 0.0f;  // the reference point of the weights, their sum
    bool ok = true;
#pragma unroll 1
    for (int j = 0; j < nt; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(&s_full[t], j & 1, abort_flag))) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t x[128];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        tmem_ld_32x32b_x32(t_lane + s_col + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&x[c * 32]));
      tmem_ld_wait();
      const int rel = lim - (jb + j) * 128;  // visible keys of the block, from its first
      if (sl < 0.0f) {
#pragma unroll
        for (int i = 0; i < 128; ++i) x[i] ^= 0x80000000u;
      }
      if (__any_sync(0xffffffffu, rel < 128)) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i >= rel) x[i] = 0xff800000u;  // -inf
      }
      float mx4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) mx4[i] = __uint_as_float(x[i]);
#pragma unroll
      for (int i = 4; i < 128; i += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + 2 * k + 1 < 128)
            mx4[k] = max3f(mx4[k], __uint_as_float(x[i + 2 * k]), __uint_as_float(x[i + 2 * k + 1]));
      const float asl = fabsf(sl);
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * asl;
      // -inf * 0 (a scale of 0 with hidden keys) is NaN, which the comparison drops
      const bool grew = mx > m + 8.0f || (m == -INFINITY && mx > -INFINITY);
      if (__any_sync(0xffffffffu, grew)) {
        const float m_new = grew ? mx : m;
        const float alpha = grew ? ex2_approx(m - m_new) : 1.0f;
        if (j > 0) {
          const uint64_t a2 = f2pack(alpha, alpha);
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t y[32];
            tmem_ld_32x32b_x32(t_lane + o_col + c * 32, y);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 v = f2unpack(mul2(f2pack(__uint_as_float(y[i]), __uint_as_float(y[i + 1])), a2));
              y[i] = __float_as_uint(v.x);
              y[i + 1] = __float_as_uint(v.y);
            }
            tmem_st_32x32b_x32(t_lane + o_col + c * 32, y);
          }
          l *= alpha;
        }
        m = m_new;
      }
      // weights 2^(s * |scale| log2 e - m); with nothing finite so far all 0
      const float m_use = m == -INFINITY ? 0.0f : m;
      const uint64_t sl2 = f2pack(asl, asl), nm2 = f2pack(-m_use, -m_use);
      uint64_t s2[2];
      s2[0] = s2[1] = f2pack(0.0f, 0.0f);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int k = h * 64 + 2 * i;
          const float2 e = f2unpack(fma2(f2pack(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), sl2, nm2));
          const float e0 = ex2_approx(e.x), e1 = ex2_approx(e.y);
          s2[i & 1] = add2(s2[i & 1], f2pack(e0, e1));
          pk[i] = pack2(e0, e1, (T*)nullptr);
        }
        tmem_st_32x32b_x32(t_lane + s_col + h * 32, pk);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[t]);
      const float2 u = f2unpack(s2[0]), v = f2unpack(s2[1]);
      l += (u.x + u.y) + (v.x + v.y);
    }
    if (ok && nt > 0) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], (nt - 1) & 1, abort_flag));
    const int64_t row = int64_t(s.q0 + token) * p.heads_q + head;
    if (!ok) {
      if (lane == 0) rec_err(a.err, abort_flag, kDevTimeoutAccFull);
    } else {
      tc_fence_after();
      T* orow = static_cast<T*>(p.O) + (s.q0 + token) * p.o_token + head * p.o_head;
      const int64_t prow = int64_t(blockIdx.z) * p.tokens_q * p.heads_q + row;
      float* parow = a.splits > 1 ? a.part_o + prow * D : nullptr;
      const bool wide = (p.o_token | p.o_head) % 8 == 0 && reinterpret_cast<uintptr_t>(p.O) % 16 == 0;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      if (a.splits > 1 && valid) a.part_ml[prow] = make_float2(m, l);
      bool bad = false;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t y[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) y[i] = 0u;
        if (nt > 0) {
          tmem_ld_32x32b_x32(t_lane + o_col + c * 32, y);
          tmem_ld_wait();
        }
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) top = max(top, y[i] & 0x7fffffffu);
        bad = bad || top >= 0x7f800000u;
        if (!valid) continue;
        if (a.splits > 1) {
          if (l != 0.0f)
#pragma unroll
            for (int g = 0; g < 8; ++g)
              reinterpret_cast<uint4*>(parow + c * 32)[g] = make_uint4(y[4 * g], y[4 * g + 1], y[4 * g + 2], y[4 * g + 3]);
          continue;
        }
        uint32_t h[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          h[i] = l == 0.0f ? 0u
                           : pack2(__uint_as_float(y[2 * i]) * inv, __uint_as_float(y[2 * i + 1]) * inv, (T*)nullptr);
        if (wide) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
            reinterpret_cast<uint4*>(orow + c * 32)[g] = make_uint4(h[4 * g], h[4 * g + 1], h[4 * g + 2], h[4 * g + 3]);
        } else {
          uint16_t* o16 = reinterpret_cast<uint16_t*>(orow + c * 32);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            o16[2 * i] = uint16_t(h[i]);
            o16[2 * i + 1] = uint16_t(h[i] >> 16);
          }
        }
      }
      // not finite although the weights are: a value the row may not see (see above)
      bad = bad && valid && l > 0.0f && l <= 3.4028234663852886e38f;
      unsigned again = __ballot_sync(0xffffffffu, bad);
      int last_bad = -1;  // of the keys that one of them may not see
      if (again != 0)
        last_bad = seq_last_bad<T, D, Q8>(p, seq, s.k0, hk, max(__reduce_min_sync(0xffffffffu, bad ? lim : kend), jb * 128),
                                          min(kend, (jb + nt) * 128));
      again = __ballot_sync(0xffffffffu, bad && last_bad >= lim);
      while (again != 0) {
        constexpr int R = 2;  // rows that share a walk over their keys (of 4 and 8 all calls' loops were 2% slower)
        const T* q[R];
        int lims[R], from[R];
        float at[R], sums[R][D / 32];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          from[r] = again != 0 ? __ffs(again) - 1 : -1;
          again &= again - 1;
          const int src = max(from[r], 0);
          const int tok = __shfl_sync(0xffffffffu, token, src), hd = __shfl_sync(0xffffffffu, head, src);
          const int sees = min(__shfl_sync(0xffffffffu, lim, src), kend);
          lims[r] = from[r] < 0 ? 0 : sees;
          at[r] = __shfl_sync(0xffffffffu, m, src);
          q[r] = static_cast<const T*>(p.Q) + (from[r] < 0 ? 0 : (s.q0 + tok) * p.q_token + hd * p.q_head);
        }
        redo_rows<T, D, Q8, R>(p, seq, s.k0, hk, q, jb * 128, lims, at, sums);
        __syncwarp();  // behind the stores of the rows' own threads, which these replace
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int src = max(from[r], 0);
          const int tok = __shfl_sync(0xffffffffu, token, src), hd = __shfl_sync(0xffffffffu, head, src);
          const float ii = __shfl_sync(0xffffffffu, inv, src);
          if (from[r] < 0) continue;
          T* of = static_cast<T*>(p.O) + (s.q0 + tok) * p.o_token + hd * p.o_head;
          float* pf = a.part_o + (int64_t(blockIdx.z) * p.tokens_q * p.heads_q + int64_t(s.q0 + tok) * p.heads_q + hd) * D;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            if (a.splits > 1) pf[lane + 32 * i] = sums[r][i];
            else stf(of + lane + 32 * i, sums[r][i] * ii);
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ------------------------------------------------------------------ joining splits
// One warp a row: weights 2^(m_z - max m) over the splits that saw a key.
template <typename T, int D>
__global__ void __launch_bounds__(128) attention_seq_combine(const SeqProblem p, const float* part_o,
                                                             const float2* part_ml, int splits) {
  pdl_trigger();
  pdl_wait();
  const int64_t rows = int64_t(p.tokens_q) * p.heads_q;
  const int64_t row = blockIdx.x * 4LL + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const int t = int(row / p.heads_q), h = int(row - int64_t(t) * p.heads_q);
  constexpr int N = D / 32;
  T* out = static_cast<T*>(p.O) + t * p.o_token + h * p.o_head + lane * N;
  const int2 rest = seq_rest(p);
  float o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.0f;
  if (t < rest.x || t >= rest.y) {
    if (!p.zero_rest) return;
  } else {
    // 32 splits at a time, a lane each; their rows are then independent loads
    float m = -INFINITY, l = 0.0f;
    for (int base = 0; base < splits; base += 32) {
      const float2 ml = base + lane < splits ? part_ml[(base + lane) * rows + row] : make_float2(-INFINITY, 0.0f);
      float top = ml.y != 0.0f ? ml.x : -INFINITY;
#pragma unroll
      for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
      const float m_new = fmaxf(m, top);
      const float old = l == 0.0f ? 0.0f : ex2_approx(m - m_new);
      const float wgt = ml.y != 0.0f ? ex2_approx(ml.x - m_new) : 0.0f;
      float sum = wgt * ml.y;
#pragma unroll
      for (int i = 16; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
      l = fmaf(l, old, sum);
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] *= old;
      m = m_new;
      const unsigned there = __ballot_sync(0xffffffffu, ml.y != 0.0f);  // the others left no row
      const int n = min(32, splits - base);
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const float f = __shfl_sync(0xffffffffu, wgt, k);
        if (!(there >> k & 1)) continue;
        const float* src = part_o + ((base + k) * rows + row) * D + lane * N;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = fmaf(f, src[i], o[i]);
      }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = l == 0.0f ? 0.0f : o[i] * inv;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) stf(out + i, o[i]);
}

// ------------------------------------------------------------------ host
template <int FMT, int D, bool Q8>
cudaError_t launch_tile_typed(const TileParams& a, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                              int64_t tiles, cudaStream_t s) {
  using Cfg = TileCfg<D, Q8>;
  using T = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
  auto kern = attention_tile_kernel<FMT, D, Q8>;
  static unsigned long long smem_set = 0;
  cudaError_t e = set_smem_once(kern, int(Cfg::SMEM), smem_set);
  if (e != cudaSuccess) return e;
  // setmaxnreg.inc waits for registers of the block's own: the shares must fit
  // what the kernel was compiled to launch with
  static int known = 0;  // (threads may make their first calls at once)
  int regs = __atomic_load_n(&known, __ATOMIC_RELAXED);
  if (regs == 0) {
    cudaFuncAttributes fa = {};
    if ((e = cudaFuncGetAttributes(&fa, kern)) != cudaSuccess) return e;
    regs = fa.numRegs;
    __atomic_store_n(&known, regs, __ATOMIC_RELAXED);
  }
  if (Cfg::WARPS / 4 * regs < Cfg::REGS_NEED) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(tiles), unsigned(a.p.heads_kv), unsigned(a.splits));
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  apply_pdl(cfg, attr, 0);
  e = cudaLaunchKernelEx(&cfg, kern, tq, tk, tv, a);
  if (e != cudaSuccess || a.splits == 1) return e;
  cfg.gridDim = dim3(unsigned((int64_t(a.p.tokens_q) * a.p.heads_q + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, attention_seq_combine<T, D>, a.p, static_cast<const float*>(a.part_o),
                            static_cast<const float2*>(a.part_ml), a.splits);
}

int64_t tile_count(const SeqProblem& p) {
  const int64_t per = 2 * (128 / p.group);
  const int64_t most = (int64_t(p.tokens_q) + int64_t(p.batch) * (per - 1)) / per;  // of any split into p.batch lengths
  return most < p.tokens_q ? (most > 0 ? most : 1) : p.tokens_q;
}

// Blocks that share a tile's keys.  Two things bound the time, in units of the
// 2.2 us a key block takes: the longest walk of a block, and all walks over the
// SMs.  A block's beginning, end and partial result cost as much as five key
// blocks, the joining kernel two.  Lengths are on the device: the longest walk
// is taken to be as long as a sequence can be, a typical one 0.6 of it.
// 32 / 8 heads of 128, unsplit and by this rule: 64 new tokens over 16000 keys
// 253 and 54 us, over 2000 39 and 20 (24 with a page table for 131072 keys), 8 x
// 100 over 800 to 8000 keys 138 and 132, 16 x 100 over 6000 205 and 205; where
// all sequences are as long as the longest, it splits too much: 4 x 200 over
// 4000 73 and 93.
int tile_splits(const SeqProblem& p, const DeviceInfo& dev) {
  const double blocks = double(tile_count(p)) * p.heads_kv, sms = dev.num_sms;
  const double keys = ((p.table != nullptr ? p.max_keys : p.tokens_kv) + 127) / 128;
  const auto cost = [&](int n) {
    const double longest = keys / n + 5, all = blocks * (0.6 * keys + 5 * n) / sms;
    return (longest > all ? longest : all) + (n > 1 ? 2 : 0);
  };
  int best = 1;
  for (int n = 2; n <= dev.num_sms && 2 * n <= keys; ++n)
    if (cost(n) < cost(best)) best = n;
  return best;
}

}  // namespace

bool seq_tile_ok(const SeqProblem& p, int dtype, int kv_dtype) {
  if ((dtype != CMPX_F16 && dtype != CMPX_BF16) || (p.d != 64 && p.d != 128) || p.group > 128) return false;
  // masked scores are -inf, which a scale of 0 would turn into NaN
  if (!(p.scale_log2 < 0.0f || p.scale_log2 > 0.0f) || p.scale_log2 - p.scale_log2 != 0.0f) return false;
  return seq_tma_ok(p, kv_dtype) && seq_rows_ok(p.Q, p.q_token, p.tokens_q, 8) &&
         seq_rows_ok(p.Q, p.q_head, p.heads_q, 8) && p.q_head * p.group < (int64_t(1) << 38) &&
         tile_count(p) <= 0x7fffffffLL && (int64_t(p.tokens_q) * p.heads_q + 3) / 4 <= 0x7fffffffLL;
}

size_t seq_tile_workspace(const SeqProblem& p, const DeviceInfo& dev) {
  const int n = tile_splits(p, dev);
  return n == 1 ? 0 : size_t(n) * size_t(p.tokens_q) * size_t(p.heads_q) * (size_t(p.d) * 4 + 8);
}

cudaError_t launch_seq_tile(const SeqProblem& p, int dtype, int kv_dtype, void* ws, const DeviceInfo& dev, int* err,
                            cudaStream_t s) {
  const bool paged = p.table != nullptr, q8 = kv_dtype == CMPX_E4M3;
  TileParams a = {};
  a.p = p;
  a.tokens = 128 / p.group;
  a.box_rows = paged && p.page_size < 128 ? p.page_size : 128;
  a.splits = tile_splits(p, dev);
  a.part_o = static_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (a.splits == 1 ? 0 : int64_t(a.splits) * p.tokens_q * p.heads_q * p.d));
  a.err = err;
  CUtensorMap tq, tk, tv;
  const uint64_t qd[4] = {uint64_t(p.d), uint64_t(p.group), uint64_t(p.heads_kv), uint64_t(p.tokens_q)};
  const int64_t qs[3] = {p.q_head, p.q_head * p.group, p.q_token};
  const bool ok = seq_rows_map(&tq, dtype, p.Q, qd, qs, 64, uint32_t(p.group), uint32_t(a.tokens), 128) &&
                  seq_kv_maps(p, kv_dtype, a.box_rows, !q8, &tk, &tv);
  if (!ok) return cudaErrorInvalidValue;
  const int64_t tiles = tile_count(p);
  if (dtype == CMPX_F16) {
    if (p.d == 64)
      return q8 ? launch_tile_typed<0, 64, true>(a, tq, tk, tv, tiles, s) : launch_tile_typed<0, 64, false>(a, tq, tk, tv, tiles, s);
    return q8 ? launch_tile_typed<0, 128, true>(a, tq, tk, tv, tiles, s) : launch_tile_typed<0, 128, false>(a, tq, tk, tv, tiles, s);
  }
  if (p.d == 64)
    return q8 ? launch_tile_typed<1, 64, true>(a, tq, tk, tv, tiles, s) : launch_tile_typed<1, 64, false>(a, tq, tk, tv, tiles, s);
  return q8 ? launch_tile_typed<1, 128, true>(a, tq, tk, tv, tiles, s) : launch_tile_typed<1, 128, false>(a, tq, tk, tv, tiles, s);
}

}  // namespace cmpx
