// Attention of few query rows per kv head (single new tokens, grouped heads)
// over packed keys or a paged cache (cmpx_attention_seq): flash decoding,
// fp16 / bf16, head_dim 64 or 128, 16-bit or e4m3 keys and values.  No
// counterpart in the reference.
//
// Every key and value is read once for the rows of a unit, so memory is the
// bound: at 44 bytes a nanosecond and SM, 128 keys of an e4m3 cache (D = 128)
// may take 0.75 us, of a 16-bit one 1.5 us.  The products need a fraction of
// that, so warp-level matrix instructions on registers serve: no
// tensor-memory round trips in the chain, and 8-bit codes are converted in
// registers between the load and the product, where the tcgen05 kernel has to
// write them back to shared memory.
//
// The products are turned around: S^T = K Q^T and O^T = V^T P^T, with keys (or
// output columns) along the 16-wide side of m16n8k16 and query rows (token x
// head of the group) along the 8-wide one.  Eight rows waste half of what
// sixteen would, and a warp's state (D x 8 sums) leaves registers for sixteen
// warps an SM, which is what hides the latency of the strip's chain of
// dependent steps.  48 single tokens of 32 / 8 heads of 128 over 1000 to 24000
// keys in an e4m3 cache: 122-130 us (5.4-5.7 TB/s of what it has to read, 82-88%
// of the copy rate), 454 with rows along the 16-wide side.
//
// Work: units (sequence, kv head, ROWS rows) of tiles (64 or 128 keys) in one
// list, each unit's beginning and end weighted like two tiles; block c of P
// takes the places [c W / P, (c + 1) W / P) of W, so ragged lengths and few
// sequences load every SM alike, and its loads run ahead across unit borders.
// A unit that lies in one block is finished there; the pieces of the others
// (at most two a block) go to the workspace and attention_decode_combine joins
// them in order of their keys.  Where no sequence can be long, blocks take
// whole units and the second kernel is spared.
//
// The last warp loads (TMA; lane i box i, a page or the whole tile, and with
// an 8-bit cache its scales; a chunk of pages looked up ahead); the others
// take strips of 16 keys in turn, each with its own maximum and sum, and meet
// when a unit's piece ends.
//
// Weights are taken against a reference point 2^2 below the first maximum and
// moved only when a score passes it by 2^8; the division by the sum of the
// same weights cancels it.
//
// An 8-bit cache runs in fp16, where its codes are exact.  bf16 queries are
// brought into fp16's range by a power of two a row (exact for magnitudes down
// to 2^-31 of the row's largest), and key scales multiply the scores in fp32.
// Value scales 2^e multiply the weights: 2^(s - m) 2^(e - d) goes with the
// codes, and o 2^d is what the sum of 2^(s - m) divides.  d = c + shift: c of
// each row follows the largest s + e of the keys it sees, so that no scale
// overflows whatever order they come in; the warp's shift (40 either way) follows
// the scales of a strip.  As long as these stay within 2^-10 .. 2^6 of every
// row's 2^d (the warp's band), weights stay below 2^14, keep fp16's bits down to
// 2^-4, and one multiplication by an exact power of two is all that takes.  A
// strip that leaves the band moves it; one that fits into no band (scales 2^16
// apart, rows that are) has its weights in two bf16 parts, 16 bits in fp32's
// range.  A strip with values beyond the largest of the queries' type, which
// are that value to every kernel, is summed key by key in fp32: rare, and kept
// out of the way of the others (products of converted values inlined in the
// loop made 48 x 3 bf16 tokens of 32 / 8 heads over 1000 to 24000 keys take 234
// us, this way 212).  Scales of 14 binades at random make 48 single tokens take
// 202 us instead of 122, where key by key it would be 690.
//
// Values that are not finite: as in attention_tile.cu, a row whose result is
// not finite although its sum is, and that may not see one of them, is
// computed again over its visible keys.
#include <cuda_fp8.h>

#include <climits>
#include <type_traits>

#include "attention_math.cuh"
#include "attention_seq.h"
#include "ptx.cuh"

namespace cmpx {
namespace {

constexpr float kBias = 2.0f, kGrow = 8.0f;
constexpr float kNone = -3.4028234663852886e38f;  // reference point of a row without a score so far

struct DecodeParams {
  SeqProblem p;
  int box_rows;     // keys of one TMA box
  int box_lg;       // log2 of them
  int blocks;       // most blocks that share the work
  int whole;        // no unit is split: a block takes whole ones, and no second kernel runs
  int rows;         // of a unit: 8 or 16
  int keys;         // of a tile
  int most;         // weight of the list that ascending offsets can make at most
  float* part_o;    // [blocks][2][rows][D]
  float2* part_ml;  // [blocks][2][rows]
  int* joints;      // [tokens_q][heads_q]: first block, pieces << 12, row of the unit << 24 (one piece: written)
  int* err;
};

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d of 2^-d.
__device__ __forceinline__ float row_exponent(float r) { return float(127 - int(__float_as_uint(r) >> 23)); }
// An 8 x 8 matrix of 16-bit values, turned.
__device__ __forceinline__ uint32_t turn8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Tiles of one unit of a sequence (one even without keys: its rows are
// written), and units of a kv head.
__device__ __forceinline__ int unit_tiles(const DecodeParams& a, int len) { return max(1, (len + a.keys - 1) / a.keys); }
__device__ __forceinline__ int row_tiles(const DecodeParams& a, int n) {
  return (n * a.p.group + a.rows - 1) / a.rows;
}
// What a unit counts for in the list that the blocks share: its tiles and
// kUnitCost for its beginning and end (queries to load, warps to join: about
// as long as two tiles take a block), or one where no unit is split.
constexpr int kUnitCost = 2;
__device__ __forceinline__ int unit_weight(const DecodeParams& a, int nt) { return a.whole ? 1 : nt + kUnitCost; }
// Tile that place x of a unit's weight stands for: the first kUnitCost + 1
// places are the first tile's.
__device__ __forceinline__ int place_tile(const DecodeParams& a, int x) { return a.whole ? 0 : max(x - kUnitCost, 0); }
// Sum of two weights, as far as an int goes.
__device__ __forceinline__ int add_weight(int x, int y) { return int(min(uint32_t(x) + uint32_t(y), 0x7fffffffu)); }
// First place of block c: floor(c * total / used).
__device__ __forceinline__ int first_place(int c, int total, int used) {
  const int q = total / used;
  return c * q + int(int64_t(c) * (total - q * used) / used);
}

// A tile in the list.
struct Walk {
  int b, hk, rt, j;  // sequence, kv head, row tile, tile of the unit
  int nrt, nt;       // row tiles, tiles of a unit
  Seq s;
  __device__ __forceinline__ void enter(const DecodeParams& a) {
    s = seq_of(a.p, b);
    nrt = row_tiles(a, s.n);
    nt = unit_tiles(a, s.len);
  }
  // The tile at place `rel` of sequence `seq`; returns the place in its unit.
  __device__ __forceinline__ int at(const DecodeParams& a, int seq, int rel) {
    b = seq;
    enter(a);
    const int weight = unit_weight(a, nt), per_head = nrt * weight;
    hk = rel / per_head;
    rel -= hk * per_head;
    rt = rel / weight;
    j = place_tile(a, rel - rt * weight);
    return rel - rt * weight;
  }
  __device__ __forceinline__ void next_unit(const DecodeParams& a) {
    j = 0;
    if (++rt < nrt) return;
    rt = 0;
    if (++hk < a.p.heads_kv) return;
    hk = 0;
    do {
      if (++b >= a.p.batch) return;  // behind the list
      enter(a);
    } while (nrt == 0);
  }
  __device__ __forceinline__ bool is(const Walk& x) const { return b == x.b && hk == x.hk && rt == x.rt && j == x.j; }
};

// What the loading warp tells the others of a tile; one lies beside each of
// the ring's places.  (The others would need a Walk of their own: with it in
// registers they spill, and with the shared memory all taken by the ring a
// spilled register comes back from L2.)
struct alignas(16) TileInfo {
  int key;           // the tile's first key
  int len;           // keys of the sequence
  int flags;
  int piece_key;     // first key of the piece of the unit that this block has
  int b, hk, row0;   // sequence, kv head, first query row (token x head of the group)
  int q0, n, k0;     // of Seq
  int pieces;        // blocks that have one, counted from this block
  int pad;
};
constexpr int kEnds = 1;     // the piece's last tile
constexpr int kWhole = 2;    // the piece is the whole unit
constexpr int kFirst = 4;    // the unit begins in this block
constexpr int kLast = 8;     // the block's last tile
constexpr int kMissing = 8;  // from this bit on: boxes of the tile (16 at most) whose page is none, 8-bit caches

// Query row r of a unit: its token, head, and visible keys (0: no such row).
struct Row {
  int token, head, lim;
  bool valid;
};
__device__ __forceinline__ Row row_of(const SeqProblem& p, const TileInfo& w, int r) {
  const int q = w.row0 + r;
  Row x;
  x.token = q / p.group;
  x.head = w.hk * p.group + q - x.token * p.group;
  x.valid = x.token < w.n;
  x.lim = x.valid ? seq_limit(p, Seq{w.q0, w.n, w.k0, w.len}, x.token) : 0;
  return x;
}

// NB: 8-row column blocks of a unit.  One needs at most 128 registers a
// thread: two blocks of eight warps an SM (registers are dealt out for four
// warps at a time, so five-warp blocks would count as eight).  Two need 168:
// one block of twelve.
template <int D, bool Q8, int NB>
struct DecodeCfg {
  static constexpr int ROWS = 8 * NB;
  static constexpr int PER_SM = NB == 1 ? 2 : 1;
  static constexpr int WARPS = NB == 1 ? 7 : 11;       // consumers
  static constexpr int THREADS = 32 * (WARPS + 1);
  static constexpr int ROW = Q8 ? D : 2 * D;           // bytes of a key
  static constexpr int KEYS = ROW == 256 ? 64 : 128;   // of a tile
  static constexpr int HALF = KEYS * ROW;              // keys, or values, of a tile
  static constexpr int RING = 196608 / PER_SM / (2 * HALF);
  static constexpr int STAGES = RING < 8 ? RING : 8;
  static constexpr int SCALES = Q8 ? 2 * KEYS : 0;     // a tile's e8m0 bytes
  static constexpr int SLOTS = NB == 1 ? WARPS : 4;    // warps whose rows of a piece fit a place of the ring
  static_assert(SLOTS * ROWS * D * 4 <= 2 * HALF, "a piece's rows fit a place of the ring");
  static constexpr size_t SMEM = size_t(STAGES) * (2 * HALF + SCALES) + STAGES * sizeof(TileInfo) + 1024 + 256 + 2 * WARPS * ROWS * 8;
  static_assert(PER_SM * (SMEM + 1024) <= 233472, "shared memory budget");
};

// Place of row r, column d of a warp's rows: the eight rows a store
// instruction touches lie on different banks.
template <int D>
__device__ __forceinline__ int merge_at(int r, int d) {
  return r * D + (d ^ ((r >> 1 & 3) << 3));
}

template <int FMT, int D, bool Q8, int NB>
__global__ void __launch_bounds__(DecodeCfg<D, Q8, NB>::THREADS, DecodeCfg<D, Q8, NB>::PER_SM)
    attention_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                            const __grid_constant__ DecodeParams a) {
  using Cfg = DecodeCfg<D, Q8, NB>;
  using T = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
  constexpr bool BF = FMT == 1 && !Q8;  // the products' type
  constexpr int KEYS = Cfg::KEYS, STAGES = Cfg::STAGES, HALF = Cfg::HALF, WARPS = Cfg::WARPS, THREADS = Cfg::THREADS;
  constexpr int DT = D / 16;            // 16-wide steps of q . k, 16-wide tiles of the output
  // largest scale byte whose codes (448 at most) stay within T's range
  constexpr uint32_t kTopScale = FMT == 0 ? 134 : 245;
  const SeqProblem& p = a.p;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024 - (raw & 1023)) & 1023);
  uint8_t* ring = smem;                                                        // [STAGES] keys, values
  uint8_t* scales = ring + size_t(STAGES) * 2 * HALF;                          // [STAGES][2][KEYS]
  TileInfo* infos = reinterpret_cast<TileInfo*>(scales + STAGES * Cfg::SCALES);  // [STAGES]
  uint64_t* full = reinterpret_cast<uint64_t*>(infos + STAGES);
  uint64_t* empty = full + STAGES;
  uint64_t* join = empty + STAGES;  // the consumers meet
  volatile int* abort_flag = reinterpret_cast<volatile int*>(join + 1);
  int* start = const_cast<int*>(abort_flag) + 1;                               // [2][2] sequence, place in it
  int* warp_sum = start + 4;                                                   // [WARPS + 1]
  float2* ml = reinterpret_cast<float2*>(warp_sum + 13);                       // [2][WARPS][ROWS]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], WARPS);
    }
    mbar_init(join, WARPS);
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_trigger();
  pdl_wait();

  // ---- this block's share of the list.  Sequences are counted THREADS at a
  // time; `mine` (the weight of this thread's sequence) and `upto` (of all up to
  // it) stay in registers where one pass holds them all.
  int mine = 0, upto = 0;
  auto count_pass = [&](int base) -> int {
    const int b = base + int(threadIdx.x);
    mine = 0;
    if (b < p.batch) {
      const Seq s = seq_of(p, b);
      mine = row_tiles(a, s.n) * unit_weight(a, unit_tiles(a, s.len)) * p.heads_kv;
    }
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto = add_weight(upto, up);
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w <= WARPS; ++w) {
      if (w == warp) upto = add_weight(upto, all);
      all = add_weight(all, warp_sum[w]);
    }
    __syncthreads();
    return all;
  };
  int total = 0;
  for (int base = 0; base < p.batch; base += THREADS) {
    const int all = count_pass(base);
    total = add_weight(total, all);
  }
  // offsets that do not ascend may name the same tokens many times: no work
  // then (and no sum that an int cannot hold)
  if (total > a.most) total = 0;
  const int used = min(total, a.blocks);
  // the places of its first tile and of the next block's
  const int c_id = int(blockIdx.x);
  const int lo = c_id < used ? first_place(c_id, total, used) : 0;
  const int hi = c_id < used ? first_place(c_id + 1, total, used) : 0;
  for (int base = 0, before = 0; lo < hi && base < p.batch; base += THREADS) {
    int all = total;
    if (p.batch > THREADS) all = count_pass(base);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rel = (e ? hi : lo) - (before + upto - mine);
      if (rel >= 0 && rel < mine) {
        start[2 * e] = base + int(threadIdx.x);
        start[2 * e + 1] = rel;
      }
    }
    before += all;
    if (hi < before) break;
  }
  __syncthreads();
  bool busy = lo < hi;
  Walk w = {}, end = {};
  int unit0 = 0;  // the unit's first place
  if (busy) {
    unit0 = lo - w.at(a, start[0], start[1]);
    end.b = p.batch;
    if (hi < total) end.at(a, start[2], start[3]);
    busy = !w.is(end);
  }

  if (warp == WARPS) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
    const int boxes_full = KEYS / a.box_rows;
    // Pages of the unit's keys, 32 at a time, a lane each: the tiles of 32
    // pages take theirs by shuffles, and the next 32 (of this unit or the
    // next one) are on their way meanwhile.
    auto pages_of = [&](const Walk& x, int chunk) -> int {
      const int at = chunk * 32 + lane;
      return p.table != nullptr && (int64_t(at) << p.page_lg) < x.s.len ? __ldg(p.table + x.b * p.table_stride + at) : 0;
    };
    int chunk = -1, page32 = 0, next32 = 0;
    if (busy) next32 = pages_of(w, (w.j * KEYS) >> p.page_lg >> 5);
    int st = 0, piece_key = w.j * KEYS;
    uint32_t phase = 1;
    int done = 0;
    bool ok = true, begins = true, last = !busy;
    while (!last) {
      const int first = (w.j * KEYS) >> p.page_lg;  // page of the tile's first key
      if (begins || first >> 5 != chunk) {
        chunk = first >> 5;
        page32 = next32;
        if ((int64_t(chunk + 1) << p.page_lg << 5) < w.s.len) {
          next32 = pages_of(w, chunk + 1);
        } else {
          Walk x = w;
          x.next_unit(a);
          if (x.b < p.batch) next32 = pages_of(x, 0);
        }
        if (begins) {
          // the queries' way from memory begins before the tile's own: a
          // 128-byte line a lane, rows of a unit in turn
          constexpr int LINES = D * 2 / 128;
          const int q = w.rt * a.rows + lane / LINES, token = q / p.group;
          if (lane < a.rows * LINES && token < w.s.n) {
            const T* at = static_cast<const T*>(p.Q) + int64_t(w.s.q0 + token) * p.q_token +
                          int64_t(w.hk * p.group + q - token * p.group) * p.q_head + lane % LINES * 64;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
          }
        }
      }
      const int now = __shfl_sync(0xffffffffu, page32, first + lane);  // (modulo 32)
      const int hk = w.hk, kv0 = w.j * KEYS, k0 = w.s.k0;
      TileInfo info;
      info.key = kv0;
      info.len = w.s.len;
      info.piece_key = piece_key;
      info.b = w.b;
      info.hk = hk;
      info.row0 = w.rt * a.rows;
      info.q0 = w.s.q0;
      info.n = w.s.n;
      info.k0 = k0;
      const int boxes = min(boxes_full, (w.s.len - kv0 + a.box_rows - 1) / a.box_rows);
      const bool unit_ends = w.j + 1 == w.nt;
      const int unit_end = unit0 + unit_weight(a, w.nt);
      if (unit_ends) {
        w.next_unit(a);
        unit0 = unit_end;
      } else {
        ++w.j;
      }
      last = w.is(end) || w.b >= p.batch;
      // blocks that hold a piece of the unit, where this is not its last tile:
      // up to the one that holds its last place, the last c with
      // c * total / used <= place
      info.pieces = 1;
      if (last && !unit_ends)
        info.pieces = min(int((int64_t(unit_end) * used - 1) / total), used - 1) - int(blockIdx.x) + 1;
      info.flags = (unit_ends || last ? kEnds : 0) | (piece_key == 0 ? kFirst : 0) |
                   (piece_key == 0 && unit_ends ? kWhole : 0) | (last ? kLast : 0);
      begins = unit_ends;
      if (unit_ends) piece_key = 0;
      if (!__all_sync(0xffffffffu, mbar_wait(&empty[st], phase, abort_flag))) {
        if (lane == 0) rec_err(a.err, abort_flag, kDevTimeoutEmpty);
        ok = false;
        break;
      }
      // pages that are none: TMA gives zeros for their codes; keys' scales 1,
      // values' 2^-127, which no band takes and a multiplication makes 0
      const bool there = lane < boxes && now >= 0 && now < p.pages;
      uint32_t bytes = uint32_t(max(boxes, 0) * a.box_rows * Cfg::ROW * 2);
      if constexpr (Q8) {
        if (lane < boxes && !there) {
          for (int k = 0; k < a.box_rows; k += 4)
#pragma unroll
            for (int v = 0; v < 2; ++v)
              *reinterpret_cast<uint32_t*>(scales + st * Cfg::SCALES + v * KEYS + lane * a.box_rows + k) =
                  v ? 0u : 0x7f7f7f7fu;
          fence_proxy_async_smem();  // before a later copy writes the place
        }
        info.flags |= int(__ballot_sync(0xffffffffu, lane < boxes && !there)) << kMissing;
        bytes += uint32_t(__popc(__ballot_sync(0xffffffffu, there)) * a.box_rows * 2);
      }
      __syncwarp();
      if (lane == 0) {
        infos[st] = info;
        mbar_arrive_expect_tx(&full[st], bytes);
      }
      __syncwarp();
      if (lane < boxes) {
        uint8_t* kd = ring + size_t(st) * 2 * HALF;
        const int row = p.table != nullptr ? (kv0 + lane * a.box_rows) & (p.page_size - 1) : k0 + kv0;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const CUtensorMap* m = v ? &tmV : &tmK;
          uint8_t* dst = kd + v * HALF;
          if constexpr (Cfg::ROW <= 128) {
            tma_load_4d(dst + lane * a.box_rows * Cfg::ROW, m, &full[st], 0, row, hk, now);
          } else {
#pragma unroll
            for (int c = 0; c < 2; ++c)
              tma_load_4d(dst + c * (HALF / 2) + lane * a.box_rows * 128, m, &full[st], c * 64, row, hk, now);
          }
          if constexpr (Q8) {
            const SeqKV& kv = v ? p.v : p.k;
            if (there)
              bulk_load(scales + st * Cfg::SCALES + v * KEYS + lane * a.box_rows,
                        kv.scale + now * kv.s_page + hk * kv.s_head + row, uint32_t(a.box_rows), &full[st]);
          }
        }
      }
      ++done;
      if (++st == STAGES) {
        st = 0;
        phase ^= 1u;
      }
    }
    if (!ok && lane == 0) {
      // let the copies in flight land before the block exits (bounded waits)
      volatile int never = 0;
      for (int i = done > STAGES ? done - STAGES : 0; i < done; ++i)
        mbar_wait(&full[i % STAGES], uint32_t((i / STAGES) & 1), &never);
    }
  } else {
    // ------------------------------------------------------------ products and softmax
    const int g = lane >> 2, t = lane & 3;
    // 16-byte unit u of strip row r lies at r * row bytes + ((u ^ swizzle) << 4);
    // this lane's row and unit of a 16 x 2-unit ldmatrix, whose four parts are
    // (rows 0-7, unit 0), (rows 8-15, unit 0), (rows 0-7, unit 1), (rows 8-15, unit 1)
    uint32_t lane_at;
    {
      const int row = (lane >> 3 & 1) * 8 + (lane & 7), unit = lane >> 4;
      constexpr int PITCH = Cfg::ROW < 128 ? 64 : 128;
      lane_at = row * PITCH + ((unit ^ (PITCH == 64 ? row >> 1 & 3 : row & 7)) << 4);
    }
    // units 2 i and 2 i + 1 of the strip at `base`
    auto ldsm_at = [&](uint32_t base, int i) -> uint32_t {
      if constexpr (Cfg::ROW == 256) return (base ^ ((2 * i & 7) << 4)) + (i >> 2) * (HALF / 2);
      else return base ^ (2 * i << 4);
    };
    constexpr int PITCH = Cfg::ROW < 128 ? 64 : 128;
    // 8-bit code of strip row j, column d (the swizzle of lane_at)
    auto code_at = [](const uint8_t* base, int j, int d) -> const uint8_t* {
      return base + j * PITCH + (((d >> 4) ^ (PITCH == 64 ? j >> 1 & 3 : j & 7)) << 4) + (d & 15);
    };
    int strip = warp;                     // the next of this warp's strips, counted from the tile's first
    int st = 0, flags = busy ? 0 : kLast;
    uint32_t phase = 0, join_phase = 0;
    int piece = 0;
    bool ok = true;
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(join);
      ok = __all_sync(0xffffffffu, mbar_wait(join, join_phase, abort_flag)) && ok;
      join_phase ^= 1u;
    };
    auto next_tile = [&]() {
      ok = __all_sync(0xffffffffu, mbar_wait(&full[st], phase, abort_flag));
      if (ok) flags = infos[st].flags;
    };
    auto release = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (++st == STAGES) {
        st = 0;
        phase ^= 1u;
      }
    };
    while (!(flags & kLast)) {  // a piece of a unit
      next_tile();
      if (!ok) break;
      uint32_t qf[DT][NB][2];               // Q^T: row g of block nb
      float o[DT][NB][4];                   // O^T: two columns, rows 2t and 2t + 1
      float m[NB][2], l[NB][2], qs[NB][2];  // rows 2t, 2t + 1: reference point, sum (this lane's keys), score factor
      float rs[NB][2];                      // 8-bit: 2^-d of the rows
      uint32_t band = 256, band_n = 0;      // 8-bit: the value scale bytes band .. band + band_n are within it (none)
      int shift = 0;                        // 8-bit: d - c of all rows
      int lim[NB][2];
      int lim_min;                          // of all rows
      {
        const TileInfo& info = infos[st];
        lim_min = info.len;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const Row r = row_of(p, info, 8 * nb + g);
          const T* q = static_cast<const T*>(p.Q) + int64_t(info.q0 + r.token) * p.q_token + r.head * p.q_head;
          float up = 1.0f;
          if constexpr (!Q8) {
#pragma unroll
            for (int k = 0; k < DT; ++k)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                qf[k][nb][e] = r.valid ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 8 * e + 2 * t) : 0u;
          } else {
            // the codes of a key arrive four consecutive ones a lane, so the
            // products' inner index is dealt out the same way
#pragma unroll
            for (int k = 0; k < DT; ++k) {
              const uint2 x = r.valid ? *reinterpret_cast<const uint2*>(q + 16 * k + 4 * t) : make_uint2(0u, 0u);
              qf[k][nb][0] = x.x;
              qf[k][nb][1] = x.y;
            }
            if constexpr (FMT == 1) {
              uint32_t top = 0;  // largest finite magnitude, as bf16 bits
#pragma unroll
              for (int k = 0; k < DT; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const uint32_t a0 = qf[k][nb][e] & 0x7fffu, a1 = qf[k][nb][e] >> 16 & 0x7fffu;
                  top = max(top, max(a0 < 0x7f80u ? a0 : 0u, a1 < 0x7f80u ? a1 : 0u));
                }
              top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
              top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
              // the row times 2^(14 - k), 2^k <= top < 2^(k + 1): below 2^15
              const float down = __uint_as_float(min(268u - (top >> 7), 254u) << 23);
              up = 1.0f / down;
#pragma unroll
              for (int k = 0; k < DT; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  qf[k][nb][e] = pack2(__uint_as_float(qf[k][nb][e] << 16) * down,
                                       __uint_as_float(qf[k][nb][e] & 0xffff0000u) * down, (__half*)nullptr);
            }
          }
          const int keys = r.valid ? r.lim : info.len;  // rows of nothing hide nothing
          lim_min = min(lim_min, __reduce_min_sync(0xffffffffu, keys));
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            qs[nb][e] = FMT == 1 && Q8 ? p.scale_log2 * __shfl_sync(0xffffffffu, up, 4 * (2 * t + e)) : p.scale_log2;
            lim[nb][e] = __shfl_sync(0xffffffffu, keys, 4 * (2 * t + e));
            m[nb][e] = kNone;
            rs[nb][e] = 1.0f;
            l[nb][e] = 0.0f;
          }
        }
#pragma unroll
        for (int k = 0; k < DT; ++k)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[k][nb][e] = 0.0f;
      }
      while (true) {  // a tile
#pragma unroll 1
        for (; strip < KEYS / 16; strip += WARPS) {
          const int kv0 = infos[st].key + strip * 16;
          const int tail = infos[st].len - kv0;  // keys of the strip
          if (tail <= 0) continue;
          const uint32_t kbase = smem_u32(ring) + st * 2 * HALF + strip * 16 * PITCH + lane_at, vbase = kbase + HALF;
          // ---- scores: keys g and g + 8, rows 2t and 2t + 1; even and odd
          // steps in chains of their own
          float s2[2][NB][4];
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int e = 0; e < 4; ++e) s2[c][nb][e] = 0.0f;
          if constexpr (!Q8) {
#pragma unroll
            for (int k = 0; k < DT; ++k) {
              uint32_t b[4];
              ldsm_x4(b, ldsm_at(kbase, k));
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) mma16<BF>(s2[k & 1][nb], b, qf[k][nb][0], qf[k][nb][1]);
            }
          } else {
#pragma unroll
            for (int k = 0; k < DT; k += 2) {
              uint32_t b[4];  // keys 0-7 and 8-15 of units k and k + 1
              ldsm_x4(b, ldsm_at(kbase, k / 2));
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                uint32_t f[4];
                e4m3_to_half(b[2 * u], f[0], f[2]);
                e4m3_to_half(b[2 * u + 1], f[1], f[3]);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mma16<false>(s2[u][nb], f, qf[k + u][nb][0], qf[k + u][nb][1]);
              }
            }
          }
          const uint8_t* sc = scales + st * Cfg::SCALES + strip * 16;
          const uint8_t* kstrip = ring + size_t(st) * 2 * HALF + strip * 16 * PITCH;  // (8-bit) its codes
          float ks[2] = {1.0f, 1.0f}, vs[2] = {1.0f, 1.0f};  // scales of keys and values g and g + 8
          // 8-bit: the strip holds a value scale out of the band, or a key that
          // may be beyond fp16's largest value (bf16's is fp32's but for half a step)
          bool odd = false;
          if constexpr (Q8) {
            bool is[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t kb = sc[g + 8 * h], vb = sc[KEYS + g + 8 * h];
              ks[h] = FMT == 0 ? __uint_as_float(kb << 23) : e8m0_to_float(kb);  // (right unless odd)
              vs[h] = __uint_as_float(vb << 23);
              is[h] = vb - band > band_n || (FMT == 0 && kb > kTopScale);
            }
            if (tail < 16) {  // what lies behind the last key may be anything
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (g + 8 * h >= tail) {
                  vs[h] = 0.0f;
                  is[h] = false;
                }
            }
            // (a page that is none holds zeros, whatever its scales)
            odd = !(flags >> (kMissing + (strip * 16 >> a.box_lg)) & 1) && (is[0] || is[1]);
          }
          // in log2 units; hidden scores -inf
          float s[NB][4];
          bool grew = false;
          const bool cut = kv0 + 16 > lim_min;
          auto hidden = [&](int nb, int e) -> bool { return cut && kv0 + g + 8 * (e >> 1) >= lim[nb][e & 1]; };
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[nb][e] = (s2[0][nb][e] + s2[1][nb][e]) * qs[nb][e & 1];
              if constexpr (Q8) s[nb][e] *= ks[e >> 1];
            }
            if (cut) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (hidden(nb, e)) s[nb][e] = -INFINITY;
            }
            grew = grew || fmaxf(s[nb][0], s[nb][2]) > m[nb][0] + kGrow || fmaxf(s[nb][1], s[nb][3]) > m[nb][1] + kGrow;
          }
          // 8-bit: a strip out of the band; one with values beyond T's largest
          bool exact = false, beyond = false;
          float ve[2] = {0.0f, 0.0f};
          if (__any_sync(0xffffffffu, grew || odd)) {
            if constexpr (Q8) {
              const int keys = flags >> (kMissing + (strip * 16 >> a.box_lg)) & 1 ? 0 : tail;
              uint32_t vb[2];
              bool live[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                live[h] = g + 8 * h < keys;
                vb[h] = sc[KEYS + g + 8 * h];
                ve[h] = e8m0_exponent(vb[h]);
                beyond = beyond || (live[h] && vb[h] > kTopScale);
              }
              beyond = __any_sync(0xffffffffu, beyond);
              if (FMT == 0 && __any_sync(0xffffffffu, (live[0] && sc[g] > kTopScale) || (live[1] && sc[g + 8] > kTopScale))) {
                // the scores of keys as T holds them, one by one
#pragma unroll 1
                for (int j = 0; j < min(keys, 16); ++j) {
                  const float up = e8m0_to_float(sc[j]);
                  float dot[NB];  // of row g of a block, this lane's columns
#pragma unroll
                  for (int nb = 0; nb < NB; ++nb) dot[nb] = 0.0f;
#pragma unroll
                  for (int k = 0; k < DT; ++k) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(code_at(kstrip, j, 16 * k + 4 * t));
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                      const uint32_t two = dequant2(e ? w >> 16 : w & 0xffffu, up, (T*)nullptr);
                      const float a0 = ldf(reinterpret_cast<const T*>(&two)), a1 = ldf(reinterpret_cast<const T*>(&two) + 1);
#pragma unroll
                      for (int nb = 0; nb < NB; ++nb) {
                        uint32_t two_q = qf[k][nb][e];
                        asm volatile("" : "+r"(two_q));  // (converted here, not ahead of the loop: that spills)
                        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&two_q));
                        dot[nb] = fmaf(x.y, a1, fmaf(x.x, a0, dot[nb]));
                      }
                    }
                  }
#pragma unroll
                  for (int nb = 0; nb < NB; ++nb) {
                    dot[nb] += __shfl_xor_sync(0xffffffffu, dot[nb], 1);
                    dot[nb] += __shfl_xor_sync(0xffffffffu, dot[nb], 2);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                      const float x = __shfl_sync(0xffffffffu, dot[nb], 4 * (2 * t + e)) * qs[nb][e];
#pragma unroll
                      for (int h = 0; h < 2; ++h)
                        if (j == g + 8 * h) s[nb][e + 2 * h] = hidden(nb, e + 2 * h) ? -INFINITY : x;
                    }
                  }
                }
              }
              // scale exponents of the strip, and of the rows that have seen a key
              int v_min = INT_MAX, v_max = INT_MIN, c_min = INT_MAX, c_max = INT_MIN;
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (live[h] && vb[h] != 255) {
                  v_min = min(v_min, int(vb[h]) - 127);
                  v_max = max(v_max, int(vb[h]) - 127);
                }
              float by[NB][2];  // exponent that the sums of a row get
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float mx = fmaxf(s[nb][e], s[nb][e + 2]);
#pragma unroll
                  for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                  const bool up = mx > m[nb][e] + kGrow;
                  const float m_new = up ? mx - kBias : m[nb][e];
                  const float d = row_exponent(rs[nb][e]), c_old = d - float(shift);
                  // largest exponent of a visible key's weight times scale, and
                  // whether one beyond the band has a weight that c must follow
                  // (-inf and NaN drop out of both; pages that are none do not count)
                  float high = -INFINITY;
                  bool over = false;
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    if (!live[h] || hidden(nb, e + 2 * h)) continue;
                    const float x = s[nb][e + 2 * h] - m_new + ve[h];
                    high = fmaxf(high, x);
                    over = over || (ve[h] - d > 6.0f && x - c_old > kGrow);
                  }
                  over = over || up;
#pragma unroll
                  for (int x = 4; x < 32; x <<= 1) {
                    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, x));
                    over = __shfl_xor_sync(0xffffffffu, int(over), x) != 0 || over;
                  }
                  const float top = fmaxf(m[nb][e] - m_new + c_old, high - kBias);
                  const float c_new = over ? fminf(fmaxf(rintf(top), -80.0f), 80.0f) : c_old;
                  l[nb][e] *= up ? ex2_approx(m[nb][e] - m_new) : 1.0f;
                  by[nb][e] = m[nb][e] - m_new + d - c_new;
                  m[nb][e] = m_new;
                  rs[nb][e] = c_new;  // (2^-d below)
                  if (m_new != kNone) {
                    c_min = min(c_min, int(c_new));
                    c_max = max(c_max, int(c_new));
                  }
                }
              v_min = __reduce_min_sync(0xffffffffu, v_min);
              v_max = __reduce_max_sync(0xffffffffu, v_max);
              c_min = __reduce_min_sync(0xffffffffu, c_min);
              c_max = __reduce_max_sync(0xffffffffu, c_max);
              const bool some = c_min <= c_max;
              if (!some) c_min = c_max = 0;
              auto fits = [&](int x) -> bool { return c_max + x - 10 <= v_min && c_min + x + 6 >= v_max; };
              if (some && v_min <= v_max && !fits(shift)) {
                const int to = max(-40, min(40, v_max - c_max));
                if (fits(to)) shift = to;
              }
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int d = int(rs[nb][e]) + shift;
                  const float alpha = ex2_approx(by[nb][e] - float(shift));
                  rs[nb][e] = __uint_as_float(uint32_t(127 - d) << 23);
#pragma unroll
                  for (int k = 0; k < DT; ++k) {
                    o[k][nb][e] *= alpha;
                    o[k][nb][e + 2] *= alpha;
                  }
                }
              const int from = max(c_max + shift + 117, 1), to = min(c_min + shift + 133, int(kTopScale));
              band = some && from <= to ? uint32_t(from) : 256u;
              band_n = some && from <= to ? uint32_t(to - from) : 0u;
              exact = __any_sync(0xffffffffu, (live[0] && vb[0] - band > band_n) || (live[1] && vb[1] - band > band_n));
            } else {
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float mx = fmaxf(s[nb][e], s[nb][e + 2]);
#pragma unroll
                  for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                  const bool up = mx > m[nb][e] + kGrow;
                  const float m_new = up ? mx - kBias : m[nb][e];
                  const float alpha = up ? ex2_approx(m[nb][e] - m_new) : 1.0f;
                  m[nb][e] = m_new;
                  l[nb][e] *= alpha;
#pragma unroll
                  for (int k = 0; k < DT; ++k) {
                    o[k][nb][e] *= alpha;
                    o[k][nb][e + 2] *= alpha;
                  }
                }
            }
          }
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = s[nb][e] - m[nb][e & 1], w = ex2_approx(x);
              l[nb][e & 1] += w;
              s[nb][e] = Q8 ? w * (vs[e >> 1] * rs[nb][e & 1]) : w;
              if (Q8 && exact)  // (w may be 0 where the scale makes up for it)
                s[nb][e] = hidden(nb, e) ? 0.0f : ex2_approx(x + (ve[e >> 1] - row_exponent(rs[nb][e & 1])));
            }
          // ---- O^T += V^T P^T.  Value rows behind the last key may hold
          // anything: their elements are cleared
          auto keep = [&](int h) -> uint32_t {
            return (8 * h + 2 * t < tail ? 0xffffu : 0u) | (8 * h + 2 * t + 1 < tail ? 0xffff0000u : 0u);
          };
          if constexpr (!Q8) {
            auto add = [&](auto clear) {
              uint32_t pf[NB][2];
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int h = 0; h < 2; ++h) pf[nb][h] = turn8x8(pack2(s[nb][2 * h], s[nb][2 * h + 1], (T*)nullptr));
#pragma unroll
              for (int k = 0; k < DT; ++k) {
                uint32_t b[4];
                ldsm_x4_t(b, ldsm_at(vbase, k));
                uint32_t f[4] = {b[0], b[2], b[1], b[3]};
                if constexpr (decltype(clear)::value) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) f[e] &= keep(e >> 1);
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mma16<BF>(o[k][nb], f, pf[nb][0], pf[nb][1]);
              }
            };
            if (tail < 16) add(std::true_type());
            else add(std::false_type());
          } else {
            // two: weights in two bf16 parts
            auto add = [&](auto two, auto clear) {
              using P = typename std::conditional<decltype(two)::value, __nv_bfloat16, __half>::type;
              uint32_t pf[NB][2], pl[NB][2];
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint32_t w = pack2(s[nb][2 * h], s[nb][2 * h + 1], (P*)nullptr);
                  pf[nb][h] = turn8x8(w);
                  if constexpr (decltype(two)::value)
                    pl[nb][h] = turn8x8(pack2(s[nb][2 * h] - __uint_as_float(w << 16),
                                              s[nb][2 * h + 1] - __uint_as_float(w & 0xffff0000u), (P*)nullptr));
                }
#pragma unroll
              for (int k = 0; k < DT; k += 2) {
                uint32_t b[4];  // units k and k + 1, each keys 0-7 and 8-15
                ldsm_x4_t(b, ldsm_at(vbase, k / 2));
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  // codes of two keys: even columns (rows 0-7 of the 16-wide
                  // side) together, and odd ones
                  uint32_t f[4];
                  e4m3_to_half(__byte_perm(b[2 * u], 0, 0x3120), f[0], f[1]);
                  e4m3_to_half(__byte_perm(b[2 * u + 1], 0, 0x3120), f[2], f[3]);
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    if constexpr (decltype(two)::value) f[e] = half2_to_bf16(f[e]);
                    if constexpr (decltype(clear)::value) f[e] &= keep(e >> 1);
                  }
#pragma unroll
                  for (int nb = 0; nb < NB; ++nb) {
                    mma16<decltype(two)::value>(o[k + u][nb], f, pf[nb][0], pf[nb][1]);
                    if constexpr (decltype(two)::value) mma16<true>(o[k + u][nb], f, pl[nb][0], pl[nb][1]);
                  }
                }
              }
            };
            if (exact && !beyond) {
              add(std::true_type(), std::true_type());
            } else if (exact) {
#pragma unroll 1
              for (int j = 0; j < min(tail, 16); ++j) {
                float w[NB][2];  // of key j, rows 2t and 2t + 1
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    w[nb][e] = __shfl_sync(0xffffffffu, j < 8 ? s[nb][e] : s[nb][e + 2], 4 * (j & 7) + t);
                const CodeScale by = code_scale(sc[KEYS + j]);
#pragma unroll
                for (int k = 0; k < DT; ++k) {
                  const uint32_t codes2 = *reinterpret_cast<const uint16_t*>(code_at(kstrip + HALF, j, 16 * k + 2 * g));
                  const uint32_t two = dequant2(codes2, by.up, (T*)nullptr);
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const float v = ldf(reinterpret_cast<const T*>(&two) + h) * by.down;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                      for (int e = 0; e < 2; ++e) o[k][nb][e + 2 * h] = fmaf(w[nb][e], v, o[k][nb][e + 2 * h]);
                  }
                }
              }
            } else if (tail < 16) {
              add(std::false_type(), std::true_type());
            } else {
              add(std::false_type(), std::false_type());
            }
          }
        }
        strip -= KEYS / 16;
        if (flags & kEnds) break;
        release();
        next_tile();
        if (!ok) break;
      }
      if (!ok) break;
      {
        const TileInfo& info = infos[st];
        // ---- join the warps: maxima and sums, then SLOTS warps' rows at a
        // time through the place of the ring whose tile was the piece's last
        // (nobody reads it any more once all have met), added in the warps'
        // order.  The maxima and sums of two pieces alternate between two
        // places: a warp may be one piece ahead of another, not two.
        constexpr int ROWS = Cfg::ROWS, SLOTS = Cfg::SLOTS, RPW = (ROWS + WARPS - 1) / WARPS;
        float2* mls = ml + piece * WARPS * ROWS;
        piece ^= 1;
        float* slots = reinterpret_cast<float*>(ring + size_t(st) * 2 * HALF);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (Q8) {
              // times 2^d; and against m + kBias, for which a single key has
              // the weight 1: its value may be the largest there is
              m[nb][e] += kBias;
              l[nb][e] *= ex2_approx(-kBias);
              const float up = ex2_approx(-kBias) * __uint_as_float((254u - (__float_as_uint(rs[nb][e]) >> 23)) << 23);
#pragma unroll
              for (int k = 0; k < DT; ++k) {
                o[k][nb][e] *= up;
                o[k][nb][e + 2] *= up;
              }
            }
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[nb][e] += __shfl_xor_sync(0xffffffffu, l[nb][e], x);
            if (g == 0) mls[warp * ROWS + 8 * nb + 2 * t + e] = make_float2(m[nb][e], l[nb][e]);
          }
        meet();
        float2 tot[RPW];   // of the rows this warp writes: warp, warp + WARPS, ...
        float acc[RPW][D / 32];
#pragma unroll
        for (int y = 0; y < RPW; ++y) {
          tot[y] = make_float2(kNone, 0.0f);
          const int r = min(warp + y * WARPS, ROWS - 1);
#pragma unroll
          for (int x = 0; x < WARPS; ++x) {
            const float2 z = mls[x * ROWS + r];
            if (z.y != 0.0f) tot[y].x = fmaxf(tot[y].x, z.x);
          }
#pragma unroll
          for (int c = 0; c < D / 32; ++c) acc[y][c] = 0.0f;
        }
#pragma unroll 1
        for (int pass = 0; pass < WARPS; pass += SLOTS) {
          if (warp >= pass && warp < pass + SLOTS) {
            float* mine = slots + (warp - pass) * ROWS * D;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int k = 0; k < DT; ++k)
#pragma unroll
                  for (int h = 0; h < 2; ++h)
                    mine[merge_at<D>(8 * nb + 2 * t + e, 16 * k + (Q8 ? 2 * g + h : g + 8 * h))] = o[k][nb][e + 2 * h];
          }
          meet();
#pragma unroll
          for (int y = 0; y < RPW; ++y) {
            const int r = min(warp + y * WARPS, ROWS - 1);
#pragma unroll
            for (int x = 0; x < SLOTS; ++x) {
              if (pass + x >= WARPS) break;
              const float2 z = mls[(pass + x) * ROWS + r];
              if (z.y == 0.0f) continue;  // saw no key: its sums are 0 times what may be anything
              const float f = ex2_approx(z.x - tot[y].x);
              tot[y].y = fmaf(z.y, f, tot[y].y);
#pragma unroll
              for (int c = 0; c < D / 32; ++c)
                acc[y][c] = fmaf(slots[x * ROWS * D + merge_at<D>(r, lane + 32 * c)], f, acc[y][c]);
            }
          }
          if (pass + SLOTS < WARPS) meet();
        }
        // ---- write out, a warp a row
#pragma unroll
        for (int y = 0; y < RPW; ++y) {
          const int r = warp + y * WARPS;
          if (r >= ROWS || !ok) continue;
          const Row row = row_of(p, info, r);
          bool bad = false;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) bad = bad || (__float_as_uint(acc[y][c]) & 0x7fffffffu) >= 0x7f800000u;
          if (!row.valid) continue;
          // the unit's first block says where its pieces lie
          if (!a.whole && (flags & kFirst) && lane == 0)
            a.joints[int64_t(info.q0 + row.token) * p.heads_q + row.head] =
                int(blockIdx.x) | info.pieces << 12 | r << 24;
          if (__any_sync(0xffffffffu, bad) && tot[y].y > 0.0f && tot[y].y <= 3.4028234663852886e38f &&
              seq_last_bad<T, D, Q8>(p, info.b, info.k0, info.hk, max(row.lim, info.piece_key),
                                     min(info.len, info.key + KEYS)) >= 0) {
            const T* const q[1] = {static_cast<const T*>(p.Q) + int64_t(info.q0 + row.token) * p.q_token +
                                   row.head * p.q_head};
            const int lims[1] = {min(row.lim, info.key + KEYS)};
            const float at[1] = {tot[y].x};
            float sums[1][D / 32];
            redo_rows<T, D, Q8, 1>(p, info.b, info.k0, info.hk, q, info.piece_key, lims, at, sums);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) acc[y][c] = sums[0][c];
          }
          if (flags & kWhole) {
            const float inv = tot[y].y == 0.0f ? 0.0f : 1.0f / tot[y].y;
            T* out = static_cast<T*>(p.O) + int64_t(info.q0 + row.token) * p.o_token + row.head * p.o_head + lane;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) stf(out + 32 * c, tot[y].y == 0.0f ? 0.0f : acc[y][c] * inv);
          } else {
            // a piece of a unit that began in an earlier block goes to the
            // first place, one that goes on in the next block to the second
            const int64_t at = (int64_t(blockIdx.x) * 2 + (flags & kFirst ? 1 : 0)) * ROWS + r;
            if (lane == 0) a.part_ml[at] = tot[y];
#pragma unroll
            for (int c = 0; c < D / 32; ++c) a.part_o[at * D + lane + 32 * c] = acc[y][c];
          }
        }
        fence_proxy_async_smem();  // before TMA writes the place again
      }
      release();
    }
    if (!ok && lane == 0) rec_err(a.err, abort_flag, kDevTimeoutFull);
  }
  // rows outside every sequence (else the joining kernel's)
  if (p.zero_rest && a.whole) {
    const int2 rest = seq_rest(p);
    const int64_t row_len = int64_t(p.heads_q) * D;
    for (int tok = blockIdx.x; tok < p.tokens_q; tok += gridDim.x)
      if (tok < rest.x || tok >= rest.y)
        for (int i = threadIdx.x; i < row_len; i += THREADS)
          stf(static_cast<T*>(p.O) + int64_t(tok) * p.o_token + (i / D) * p.o_head + i % D, 0.0f);
  }
}

// Joins the pieces of units that span blocks: one warp a (token, head).
template <typename T, int D>
__global__ void __launch_bounds__(128) attention_decode_combine(const DecodeParams a) {
  const SeqProblem& p = a.p;
  pdl_trigger();
  pdl_wait();
  const int64_t row = blockIdx.x * 4LL + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= int64_t(p.tokens_q) * p.heads_q) return;
  const int t = int(row / p.heads_q), h = int(row - int64_t(t) * p.heads_q);
  constexpr int N = D / 32;
  T* out = static_cast<T*>(p.O) + int64_t(t) * p.o_token + h * p.o_head + lane * N;
  const int2 rest = seq_rest(p);
  if (t < rest.x || t >= rest.y) {
    if (p.zero_rest)
#pragma unroll
      for (int i = 0; i < N; ++i) stf(out + i, 0.0f);
    return;
  }
  // (clamped: offsets that are not ascending leave rows that no block wrote)
  const int joint = a.joints[row];
  const int c0 = min(joint & 0xfff, a.blocks - 1), c1 = min(c0 + (joint >> 12 & 0xfff) - 1, a.blocks - 1);
  const int r = min(joint >> 24 & 0xff, a.rows - 1);
  if (c0 >= c1) return;  // whole in one block: written there
  // the unit begins in block c0's second piece and goes on in the others' first
  auto at = [&](int c) -> int64_t { return (int64_t(c) * 2 + (c == c0 ? 1 : 0)) * a.rows + r; };
  // 32 pieces at a time, a lane each; their rows are then independent loads
  float m = kNone, l = 0.0f, o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.0f;
  for (int base = c0; base <= c1; base += 32) {
    const int64_t mine = base + lane <= c1 ? at(base + lane) : -1;
    const float2 ml = mine >= 0 ? a.part_ml[mine] : make_float2(kNone, 0.0f);
    float top = ml.y != 0.0f ? ml.x : kNone;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    const float m_new = fmaxf(m, top), old = ex2_approx(m - m_new);
    const float wgt = ml.y != 0.0f ? ex2_approx(ml.x - m_new) : 0.0f;
    float sum = wgt * ml.y;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    l = fmaf(l, old, sum);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] *= old;
    m = m_new;
    const int n = min(32, c1 - base + 1);
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float f = __shfl_sync(0xffffffffu, wgt, k);
      const float* src = a.part_o + __shfl_sync(0xffffffffu, mine, k) * D + lane * N;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = fmaf(f, src[i], o[i]);  // (a piece that saw no key holds zeros)
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < N; ++i) stf(out + i, l == 0.0f ? 0.0f : o[i] * inv);
}

// ------------------------------------------------------------------ host
int decode_keys(const SeqProblem& p, bool q8) {
  return p.d == 64 ? (q8 ? DecodeCfg<64, true, 1>::KEYS : DecodeCfg<64, false, 1>::KEYS)
                   : (q8 ? DecodeCfg<128, true, 1>::KEYS : DecodeCfg<128, false, 1>::KEYS);
}
int64_t decode_blocks(const DeviceInfo& dev, int rows) { return int64_t(dev.num_sms) * (rows == 8 ? 2 : 1); }
// Sequences that cannot be long: splitting them among blocks saves less than
// the second kernel costs.  Whole and split, 32 / 8 heads of 128, one token over
// 512 keys 11.1 and 14.3 us, over 1024 15.6 and 14.7; 16 tokens 12.7 and 16.2,
// 18.2 and 18.5; 128 tokens, which need no splitting, 62 and 54, 97 and 93.
bool decode_whole(const SeqProblem& p) { return (p.table != nullptr ? p.max_keys : p.tokens_kv) <= 512; }

// More places than any lengths can make of the problem (64 keys, 8 rows each).
double most_places(const SeqProblem& p) {
  const double rows = double(p.tokens_q) * p.group / 8 + p.batch;
  const double keys = double(p.table != nullptr ? p.max_keys : p.tokens_kv) / 64 + 1;
  return rows * (keys + kUnitCost) * p.heads_kv;
}

template <int FMT, int D, bool Q8, int NB>
cudaError_t launch_decode_rows(const DecodeParams& a, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t s) {
  using Cfg = DecodeCfg<D, Q8, NB>;
  using T = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
  auto kern = attention_decode_kernel<FMT, D, Q8, NB>;
  static unsigned long long smem_set = 0, carve_set = 0;
  cudaError_t e = set_smem_once(kern, int(Cfg::SMEM), smem_set);
  // all of the SM's shared memory, or fewer than PER_SM blocks would share it
  if (e == cudaSuccess)
    e = set_attribute_once(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared, carve_set);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.blocks));
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  apply_pdl(cfg, attr, 0);
  e = cudaLaunchKernelEx(&cfg, kern, tk, tv, a);
  if (e != cudaSuccess || a.whole) return e;
  cfg.gridDim = dim3(unsigned((int64_t(a.p.tokens_q) * a.p.heads_q + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, attention_decode_combine<T, D>, a);
}

template <int FMT, int D, bool Q8>
cudaError_t launch_decode_typed(const DecodeParams& a, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t s) {
  return a.rows == 8 ? launch_decode_rows<FMT, D, Q8, 1>(a, tk, tv, s) : launch_decode_rows<FMT, D, Q8, 2>(a, tk, tv, s);
}

}  // namespace

bool seq_decode_ok(const SeqProblem& p, int dtype, int kv_dtype) {
  return (dtype == CMPX_F16 || dtype == CMPX_BF16) && (p.d == 64 || p.d == 128) && seq_tma_ok(p, kv_dtype) &&
         seq_rows_ok(p.Q, p.q_token, p.tokens_q, 8) && seq_rows_ok(p.Q, p.q_head, p.heads_q, 8) &&
         (int64_t(p.tokens_q) * p.heads_q + 3) / 4 <= 0x7fffffffLL && most_places(p) < 0x7fffffff;
}

size_t seq_decode_workspace(const SeqProblem& p, int rows, const DeviceInfo& dev) {
  if (decode_whole(p)) return 0;
  return size_t(decode_blocks(dev, rows)) * 2 * size_t(rows) * (size_t(p.d) * 4 + 8) + size_t(p.tokens_q) * size_t(p.heads_q) * 4;
}

cudaError_t launch_seq_decode(const SeqProblem& p, int dtype, int kv_dtype, int rows, void* ws, const DeviceInfo& dev,
                              int* err, cudaStream_t s) {
  const bool paged = p.table != nullptr, q8 = kv_dtype == CMPX_E4M3;
  DecodeParams a = {};
  a.p = p;
  a.rows = rows;
  a.keys = decode_keys(p, q8);
  a.box_rows = paged && p.page_size < a.keys ? p.page_size : a.keys;
  while ((2 << a.box_lg) <= a.box_rows) ++a.box_lg;
  a.whole = decode_whole(p);
  if (a.whole) {
    // a block a unit, up to a few waves
    const int64_t units = ((int64_t(p.tokens_q) * p.group + int64_t(p.batch) * (rows - 1)) / rows) * p.heads_kv;
    const int64_t most = 8 * decode_blocks(dev, rows);
    a.blocks = int(units < 1 ? 1 : units < most ? units : most);
  } else {
    a.blocks = int(decode_blocks(dev, rows));
    a.part_o = static_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + int64_t(a.blocks) * 2 * rows * p.d);
    a.joints = reinterpret_cast<int*>(a.part_ml + int64_t(a.blocks) * 2 * rows);
  }
  a.most = int(most_places(p));
  a.err = err;
  CUtensorMap tk, tv;
  if (!seq_kv_maps(p, kv_dtype, a.box_rows, true, &tk, &tv)) return cudaErrorInvalidValue;
  if (dtype == CMPX_F16) {
    if (p.d == 64) return q8 ? launch_decode_typed<0, 64, true>(a, tk, tv, s) : launch_decode_typed<0, 64, false>(a, tk, tv, s);
    return q8 ? launch_decode_typed<0, 128, true>(a, tk, tv, s) : launch_decode_typed<0, 128, false>(a, tk, tv, s);
  }
  if (p.d == 64) return q8 ? launch_decode_typed<1, 64, true>(a, tk, tv, s) : launch_decode_typed<1, 64, false>(a, tk, tv, s);
  return q8 ? launch_decode_typed<1, 128, true>(a, tk, tv, s) : launch_decode_typed<1, 128, false>(a, tk, tv, s);
}

}  // namespace cmpx
