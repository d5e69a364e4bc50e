// Attention of few query rows per kv head (single new tokens, grouped heads)
// over packed keys or a paged cache (cmpx_attention_seq): flash decoding,
// fp16 / bf16, head_dim 64 or 128, 16-bit or e4m3 keys and values.  No
// counterpart in the reference.
//
// Every key and value is read once for 16 rows, so memory is the bound: at
// 44 bytes a nanosecond and SM, 128 keys of an e4m3 cache (D = 128) may take
// 0.75 us, of a 16-bit one 1.5 us.  The products (m16n8k16, rows = token x
// head of the group, padded to 16) need a fraction of that, so warp-level
// matrix instructions on registers serve: no tensor-memory round trips in the
// chain, and 8-bit codes are converted in registers between the load and the
// product, where the tcgen05 kernel has to write them back to shared memory.
//
// Work: units (sequence, kv head, 16 rows) of ceil(keys / 128) tiles in one
// list of W tiles; block c of P takes tiles [c W / P, (c + 1) W / P), so
// ragged lengths and few sequences load every SM alike, and its loads run
// ahead across unit borders.  A unit that lies in one block is finished
// there; the pieces of the others (at most two a block) go to the workspace
// and attention_decode_combine joins them in order of their keys.
//
// Warp 8 loads (TMA; lane i box i, a page or the whole tile; with an 8-bit
// cache also the tile's scales, as floats, a tile ahead); warps 0-7 take 16
// keys of a tile each, with their own maximum and sum, and meet when a unit's
// piece ends.
//
// Weights are taken against a reference point 2^6 below the first maximum and
// moved only when a score passes it by 2^14 (fp16 weights stay below 2^15, and
// those above 2^-14 of the top keep all their bits); the division by the sum
// of the same weights cancels it.
//
// An 8-bit cache runs in fp16: codes are exact there.  bf16 queries are
// brought into fp16's range by a power of two a row (exact for magnitudes
// down to 2^-31 of the row's largest), key scales multiply the scores in
// fp32, value scales the codes (exact while 2^-15 <= scale <= 2^7; a strip
// of 16 keys with another one goes through fp32 into the queries' type).
//
// Values that are not finite: as in attention_tile.cu, a row whose result is
// not finite although its sum is is computed again over its visible keys.
#include <cuda_fp8.h>

#include <type_traits>

#include "attention_math.cuh"
#include "attention_seq.h"
#include "ptx.cuh"

namespace cmpx {
namespace {

constexpr int kKeys = 128;        // keys of a tile
constexpr int kConsumers = 8;     // warps, 16 keys each
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr float kBias = 6.0f, kGrow = 14.0f;

template <int D, bool Q8>
struct DecodeCfg {
  static constexpr int ROW = Q8 ? D : 2 * D;           // bytes of a key
  static constexpr int HALF = kKeys * ROW;             // keys, or values, of a tile
  static constexpr int STAGES = (Q8 ? 163840 : 196608) / (2 * HALF) < 8 ? (Q8 ? 163840 : 196608) / (2 * HALF) : 8;
  static constexpr int SCALES = Q8 ? 2 * kKeys * 4 : 0;
  static constexpr int MERGE = 4 * 16 * D * 4;         // four warps' rows
  static constexpr size_t SMEM = size_t(STAGES) * (2 * HALF + SCALES) + MERGE + 1024 + 2048;
  static_assert(SMEM <= 232448, "shared memory budget");
};

struct DecodeParams {
  SeqProblem p;
  int box_rows;     // keys of one TMA box
  int blocks;       // most blocks that share the work
  int min_tiles;    // tiles worth a block
  float* part_o;    // [blocks][2][16][D]
  float2* part_ml;  // [blocks][2][16]
  int64_t* plan;    // [batch + 2]: tiles before each sequence, their number, blocks in use
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
__device__ __forceinline__ uint32_t cvt_e4m3x2(uint32_t two) {  // low 16 bits: two codes
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two), __NV_E4M3);
  return uint32_t(h.x) | uint32_t(h.y) << 16;
}
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t scaled2(uint32_t h2, float lo, float hi, __half*) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(f.y * hi), "f"(f.x * lo));
  return r;
}
__device__ __forceinline__ uint32_t scaled2(uint32_t h2, float lo, float hi, __nv_bfloat16*) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
  uint32_t r;
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(f.y * hi), "f"(f.x * lo));
  return r;
}
__device__ __forceinline__ void sync_consumers() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kConsumers) : "memory"); }

// Tiles of one unit of a sequence (one even without keys: its rows are
// written), and units of a kv head.
__device__ __forceinline__ int unit_tiles(int len) { return max(1, (len + kKeys - 1) / kKeys); }
__device__ __forceinline__ int row_tiles(int n, int group) { return (n * group + 15) >> 4; }
// First tile of block c.
__device__ __forceinline__ int64_t first_tile(int64_t c, int64_t total, int64_t used) { return c * total / used; }

// A place in the list of tiles.
struct Walk {
  int b, hk, rt, j;  // sequence, kv head, row tile, tile of the unit
  int nrt, nt;       // row tiles, tiles of a unit
  Seq s;
  __device__ __forceinline__ void enter(const SeqProblem& p) {
    s = seq_of(p, b);
    nrt = row_tiles(s.n, p.group);
    nt = unit_tiles(s.len);
  }
  __device__ __forceinline__ void step(const SeqProblem& p) {
    if (++j < nt) return;
    j = 0;
    if (++rt < nrt) return;
    rt = 0;
    if (++hk < p.heads_kv) return;
    hk = 0;
    do {
      if (++b >= p.batch) return;  // behind the list
      enter(p);
    } while (nrt == 0);
  }
};

// The row (16 of a unit) with index r: its token, head, and visible keys (0:
// no such row).
struct Row {
  int token, head, lim;
  bool valid;
};
__device__ __forceinline__ Row row_of(const SeqProblem& p, const Walk& w, int r) {
  const int q = w.rt * 16 + r;
  Row x;
  x.token = q / p.group;
  x.head = w.hk * p.group + q - x.token * p.group;
  x.valid = x.token < w.s.n;
  x.lim = x.valid ? seq_limit(p, w.s, x.token) : 0;
  return x;
}

// Place of row r, column d among a warp pair's joined rows: rows four apart
// share banks, so the eight a store instruction touches conflict two by two.
template <int D>
__device__ __forceinline__ int merge_at(int r, int d) {
  return r * D + (d ^ ((r & 3) << 3));
}

// One row over keys [kbeg, kend) from its definition; a warp computes it.
template <typename T, int D, bool Q8>
__device__ __noinline__ void redo_row(const SeqProblem& p, int b, int k0, int hk, const T* q, int kbeg, int kend,
                                      float m, float* merge, int r) {
  const int lane = threadIdx.x & 31;
  constexpr int NV = D / 32;
  using KV = typename std::conditional<Q8, __nv_fp8_e4m3, T>::type;
  auto load = [](const KV* at) -> float {
    if constexpr (Q8) return float(*at);
    else return ldf(at);
  };
  float acc[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = 0.0f;
  for (int j = kbeg; j < kend; ++j) {
    int64_t ko = int64_t(k0 + j) * p.k.row, vo = int64_t(k0 + j) * p.v.row;
    float ks = 1.0f, vs = 1.0f;
    if (p.table != nullptr) {
      const int page = __ldg(p.table + b * p.table_stride + j / p.page_size), slot = j % p.page_size;
      if (page < 0 || page >= p.pages) continue;  // zeros
      ko = page * p.k.page + slot * p.k.row;
      vo = page * p.v.page + slot * p.v.row;
      if (Q8) {
        ks = e8m0_to_float(p.k.scale[page * p.k.s_page + hk * p.k.s_head + slot * p.k.s_row]);
        vs = e8m0_to_float(p.v.scale[page * p.v.s_page + hk * p.v.s_head + slot * p.v.s_row]);
      }
    }
    const KV* kr = static_cast<const KV*>(p.k.base) + ko + hk * p.k.head;
    const KV* vr = static_cast<const KV*>(p.v.base) + vo + hk * p.v.head;
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) dot = fmaf(ldf(q + lane + 32 * i), load(kr + lane + 32 * i), dot);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float w = ex2_approx(dot * ks * p.scale_log2 - m) * vs;
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = fmaf(w, load(vr + lane + 32 * i), acc[i]);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) merge[merge_at<D>(r, lane + 32 * i)] = acc[i];
}

template <int FMT, int D, bool Q8>
__global__ void __launch_bounds__(kThreads, 1)
    attention_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                            const __grid_constant__ DecodeParams a) {
  using Cfg = DecodeCfg<D, Q8>;
  using T = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
  constexpr bool BF = FMT == 1 && !Q8;          // the products' type
  constexpr int STAGES = Cfg::STAGES, HALF = Cfg::HALF;
  constexpr int KSTEPS = D / 16, OT = D / 8;    // 16-wide steps of q . k, 8-wide tiles of the output
  const SeqProblem& p = a.p;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024 - (raw & 1023)) & 1023);
  uint8_t* ring = smem;                                                        // [STAGES] keys, values
  float* merge = reinterpret_cast<float*>(ring + size_t(STAGES) * 2 * HALF);   // [4][16][D]
  float* scales = merge + Cfg::MERGE / 4;                                      // [STAGES][2][kKeys]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + STAGES * (Cfg::SCALES / 4));
  uint64_t* empty = full + STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + STAGES);
  int* start = const_cast<int*>(abort_flag) + 2;                               // [4] sequence, then the place in it
  int64_t* warp_sum = reinterpret_cast<int64_t*>(start + 4);                   // [9]
  float2* ml = reinterpret_cast<float2*>(warp_sum + 10);                       // [8][16]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], Q8 ? 33 : 1);
      mbar_init(&empty[i], kConsumers);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_trigger();
  pdl_wait();

  // ---- this block's share of the tiles
  auto tiles_of = [&](int b) -> int64_t {
    if (b >= p.batch) return 0;
    const Seq s = seq_of(p, b);
    return int64_t(row_tiles(s.n, p.group)) * unit_tiles(s.len) * p.heads_kv;
  };
  // inclusive sum over a chunk of kThreads sequences, and the chunk's total
  auto scan = [&](int64_t c, int64_t& all) -> int64_t {
    int64_t inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int w = 0; w <= kConsumers; ++w) {
      if (w == warp) inc += all;
      all += warp_sum[w];
    }
    __syncthreads();
    return inc;
  };
  int64_t total = 0;
  for (int base = 0; base < p.batch; base += kThreads) {
    const int64_t c = tiles_of(base + int(threadIdx.x));
    int64_t all;
    const int64_t inc = scan(c, all);
    if (blockIdx.x == 0 && base + int(threadIdx.x) < p.batch)
      a.plan[base + threadIdx.x] = total + inc - c;
    total += all;
  }
  int64_t used = (total + a.min_tiles - 1) / a.min_tiles;
  if (used > a.blocks) used = a.blocks;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.plan[p.batch] = total;
    a.plan[p.batch + 1] = used;
  }
  const int64_t c_id = blockIdx.x;
  const int64_t lo = c_id < used ? first_tile(c_id, total, used) : 0;
  const int64_t hi = c_id < used ? first_tile(c_id + 1, total, used) : 0;
  int64_t before = 0;
  for (int base = 0; lo < hi && base < p.batch; base += kThreads) {
    const int64_t c = tiles_of(base + int(threadIdx.x));
    int64_t all;
    const int64_t inc = scan(c, all);
    const int64_t rel = lo - (before + inc - c);
    if (rel >= 0 && rel < c) {
      start[0] = base + int(threadIdx.x);
      *reinterpret_cast<int64_t*>(start + 2) = rel;
    }
    __syncthreads();
    before += all;
    if (lo < before) break;
  }
  Walk w = {};
  if (lo < hi) {
    w.b = start[0];
    int64_t rel = *reinterpret_cast<int64_t*>(start + 2);
    w.enter(p);
    const int64_t per_head = int64_t(w.nrt) * w.nt;
    w.hk = int(rel / per_head);
    rel -= w.hk * per_head;
    w.rt = int(rel / w.nt);
    w.j = int(rel - int64_t(w.rt) * w.nt);
  }

  if (warp == kConsumers) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      prefetch_tmap(&tmK);
      prefetch_tmap(&tmV);
    }
    const int boxes_full = kKeys / a.box_rows;
    struct Ahead {
      int page;        // of this lane's box
      float ks[4], vs[4];  // scales of keys 4 lane .. 4 lane + 3
    };
    auto look = [&](const Walk& x) -> Ahead {
      Ahead h;
      h.page = 0;
      const int kv0 = x.j * kKeys;
      if (p.table != nullptr) {
        const int key = kv0 + lane * a.box_rows;
        if (lane < boxes_full && key < x.s.len) h.page = __ldg(p.table + x.b * p.table_stride + key / p.page_size);
      }
      if constexpr (Q8) {
        const int page = __shfl_sync(0xffffffffu, h.page, (4 * lane) / a.box_rows);
        const bool there = page >= 0 && page < p.pages;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = kv0 + 4 * lane + i, slot = key & (p.page_size - 1);
          h.ks[i] = h.vs[i] = 0.0f;
          if (there && key < x.s.len) {
            h.ks[i] = e8m0_to_float(__ldg(p.k.scale + page * p.k.s_page + x.hk * p.k.s_head + slot * p.k.s_row));
            h.vs[i] = e8m0_to_float(__ldg(p.v.scale + page * p.v.s_page + x.hk * p.v.s_head + slot * p.v.s_row));
          }
        }
      }
      return h;
    };
    Ahead next = {};
    if (lo < hi) next = look(w);
    int64_t done = 0;
    bool ok = true;
    for (int64_t i = lo; i < hi; ++i) {
      const Ahead now = next;
      const int hk = w.hk, kv0 = w.j * kKeys, k0 = w.s.k0;
      const int boxes = min(boxes_full, (w.s.len - kv0 + a.box_rows - 1) / a.box_rows);
      w.step(p);
      if (i + 1 < hi) next = look(w);
      const int st = int((i - lo) % STAGES);
      if (!__all_sync(0xffffffffu, mbar_wait(&empty[st], uint32_t(((i - lo) / STAGES) & 1) ^ 1u, abort_flag))) {
        if (lane == 0) rec_err(a.err, abort_flag, kDevTimeoutEmpty);
        ok = false;
        break;
      }
      if (lane == 0) mbar_arrive_expect_tx(&full[st], uint32_t(max(boxes, 0) * a.box_rows * Cfg::ROW * 2));
      __syncwarp();
      if (lane < boxes) {
        uint8_t* kd = ring + size_t(st) * 2 * HALF;
        const int row = p.table != nullptr ? (kv0 + lane * a.box_rows) & (p.page_size - 1) : k0 + kv0;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const CUtensorMap* m = v ? &tmV : &tmK;
          uint8_t* dst = kd + v * HALF;
          if constexpr (Cfg::ROW <= 128) {
            tma_load_4d(dst + lane * a.box_rows * Cfg::ROW, m, &full[st], 0, row, hk, now.page);
          } else {
#pragma unroll
            for (int c = 0; c < 2; ++c)
              tma_load_4d(dst + c * (HALF / 2) + lane * a.box_rows * 128, m, &full[st], c * 64, row, hk, now.page);
          }
        }
      }
      if constexpr (Q8) {
        float* sc = scales + st * 2 * kKeys;
        *reinterpret_cast<float4*>(sc + 4 * lane) = make_float4(now.ks[0], now.ks[1], now.ks[2], now.ks[3]);
        *reinterpret_cast<float4*>(sc + kKeys + 4 * lane) = make_float4(now.vs[0], now.vs[1], now.vs[2], now.vs[3]);
        mbar_arrive(&full[st]);
      }
      ++done;
    }
    if (!ok && lane == 0) {
      // let the copies in flight land before the block exits (bounded waits)
      volatile int never = 0;
      for (int64_t i = done > STAGES ? done - STAGES : 0; i < done; ++i)
        mbar_wait(&full[i % STAGES], uint32_t((i / STAGES) & 1), &never);
    }
  } else {
    // ------------------------------------------------------------ products and softmax
    const int g = lane >> 2, t = lane & 3;
    const int key_w = warp * 16;  // this warp's keys of a tile
    uint32_t qf[KSTEPS][4];
    float o[OT][4];
    float m[2], l[2], qs[2];  // rows g and g + 8: reference point, sum (this lane's keys), score factor
    int lim[2] = {0, 0};
    bool fresh = true, ok = true;
    const int mi = lane >> 3, mr = lane & 7;
    for (int64_t i = lo; i < hi; ++i) {
      if (fresh) {
        fresh = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Row r = row_of(p, w, g + 8 * h);
          lim[h] = r.valid ? r.lim : w.s.len;  // rows of nothing hide nothing
          m[h] = -INFINITY;
          l[h] = 0.0f;
          qs[h] = p.scale_log2;
          const T* q = static_cast<const T*>(p.Q) + int64_t(w.s.q0 + r.token) * p.q_token + r.head * p.q_head;
          if constexpr (!Q8) {
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
              qf[k][h] = r.valid ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * t) : 0u;
              qf[k][2 + h] = r.valid ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 8 + 2 * t) : 0u;
            }
          } else {
            // the codes of a key arrive four consecutive ones a lane, so the
            // products' inner index is dealt out the same way
            uint2 x[KSTEPS];
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k)
              x[k] = r.valid ? *reinterpret_cast<const uint2*>(q + 16 * k + 4 * t) : make_uint2(0u, 0u);
            if constexpr (FMT == 1) {
              uint32_t top = 0;  // largest magnitude, as bf16 bits
#pragma unroll
              for (int k = 0; k < KSTEPS; ++k) {
                top = max(top, max(x[k].x & 0x7fffu, x[k].x >> 16 & 0x7fffu));
                top = max(top, max(x[k].y & 0x7fffu, x[k].y >> 16 & 0x7fffu));
              }
              top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
              top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
              // the row times 2^(14 - k), 2^k <= top < 2^(k + 1): below 2^15
              const int e = int(top >> 7);
              const bool plain = e == 0 || e == 255;
              const float down = plain ? 1.0f : __uint_as_float(uint32_t(min(max(127 + 14 + 127 - e, 1), 254)) << 23);
              const float up = plain ? 1.0f : 1.0f / down;
              qs[h] = p.scale_log2 * up;
#pragma unroll
              for (int k = 0; k < KSTEPS; ++k) {
                x[k].x = pack2(__uint_as_float(x[k].x << 16) * down, __uint_as_float(x[k].x & 0xffff0000u) * down,
                               (__half*)nullptr);
                x[k].y = pack2(__uint_as_float(x[k].y << 16) * down, __uint_as_float(x[k].y & 0xffff0000u) * down,
                               (__half*)nullptr);
              }
            }
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
              qf[k][h] = x[k].x;
              qf[k][2 + h] = x[k].y;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < OT; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[k][e] = 0.0f;
      }
      const int st = int((i - lo) % STAGES);
      if (ok && !__all_sync(0xffffffffu, mbar_wait(&full[st], uint32_t(((i - lo) / STAGES) & 1), abort_flag))) {
        if (lane == 0) rec_err(a.err, abort_flag, kDevTimeoutFull);
        ok = false;
      }
      const int kv0 = w.j * kKeys + key_w;
      if (ok && kv0 < w.s.len) {
        const uint32_t kbase = smem_u32(ring + size_t(st) * 2 * HALF), vbase = kbase + HALF;
        // address of 16-byte unit u of row r (128- or 64-byte swizzled rows)
        auto unit_at = [&](uint32_t base, int r, int u) -> uint32_t {
          if constexpr (Cfg::ROW == 256) return base + (u >> 3) * (HALF / 2) + r * 128 + (((u & 7) ^ (r & 7)) << 4);
          else if constexpr (Cfg::ROW == 128) return base + r * 128 + ((u ^ (r & 7)) << 4);
          else return base + r * 64 + ((u ^ (r >> 1 & 3)) << 4);
        };
        // ---- scores of 16 rows x 16 keys: two tiles of 8 keys
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
        if constexpr (!Q8) {
#pragma unroll
          for (int k = 0; k < KSTEPS; ++k) {
            uint32_t b[4];
            ldsm_x4(b, unit_at(kbase, key_w + (mi >> 1) * 8 + mr, 2 * k + (mi & 1)));
            mma16<BF>(s[0], qf[k], b[0], b[1]);
            mma16<BF>(s[1], qf[k], b[2], b[3]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < KSTEPS; k += 2) {
            uint32_t b[4];
            ldsm_x4(b, unit_at(kbase, key_w + (mi >> 1) * 8 + mr, k + (mi & 1)));
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int kk = 0; kk < 2; ++kk)
                mma16<false>(s[n], qf[k + kk], cvt_e4m3x2(b[2 * n + kk] & 0xffffu), cvt_e4m3x2(b[2 * n + kk] >> 16));
          }
        }
        // ---- scores in log2 units; hidden ones -inf
        const float* sc = scales + st * 2 * kKeys + key_w;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          float2 kf = make_float2(1.0f, 1.0f);
          if constexpr (Q8) kf = *reinterpret_cast<const float2*>(sc + 8 * n + 2 * t);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[n][e] *= qs[e >> 1];
            if constexpr (Q8) s[n][e] *= (e & 1) ? kf.y : kf.x;
          }
        }
        const int edge = min(lim[0], lim[1]) - kv0;
        const bool cut = __any_sync(0xffffffffu, edge < 16);
        if (cut) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (kv0 + 8 * n + 2 * t + (e & 1) >= lim[e >> 1]) s[n][e] = -INFINITY;
        }
        float mx[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          mx[h] = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
        const bool grew = mx[0] > m[0] + kGrow || mx[1] > m[1] + kGrow;
        if (__any_sync(0xffffffffu, grew)) {
          float alpha[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            const float m_new = mx[h] > m[h] + kGrow ? mx[h] - kBias : m[h];
            alpha[h] = m_new == m[h] ? 1.0f : ex2_approx(m[h] - m_new);
            m[h] = m_new;
            l[h] *= alpha[h];
          }
#pragma unroll
          for (int k = 0; k < OT; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[k][e] *= alpha[e >> 1];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float mu = m[h] == -INFINITY ? 0.0f : m[h];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float wgt = ex2_approx(s[n][2 * h + e] - mu);
              s[n][2 * h + e] = wgt;
              l[h] += wgt;
            }
        }
        // ---- O += P V
        const int tail = w.s.len - kv0;  // keys of the strip
        // value rows behind the last key may hold anything: lanes clear theirs
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
        if (tail < 16) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            keep[h] = (8 * h + 2 * t < tail ? 0xffffu : 0u) | (8 * h + 2 * t + 1 < tail ? 0xffff0000u : 0u);
        }
        if constexpr (!Q8) {
          const uint32_t pf[4] = {pack2(s[0][0], s[0][1], (T*)nullptr), pack2(s[0][2], s[0][3], (T*)nullptr),
                                  pack2(s[1][0], s[1][1], (T*)nullptr), pack2(s[1][2], s[1][3], (T*)nullptr)};
#pragma unroll
          for (int k = 0; k < OT; k += 2) {
            uint32_t b[4];
            ldsm_x4_t(b, unit_at(vbase, key_w + (mi & 1) * 8 + mr, k + (mi >> 1)));
            mma16<BF>(o[k], pf, b[0] & keep[0], b[1] & keep[1]);
            mma16<BF>(o[k + 1], pf, b[2] & keep[0], b[3] & keep[1]);
          }
        } else {
          const float2 v0 = *reinterpret_cast<const float2*>(sc + kKeys + 2 * t);
          const float2 v1 = *reinterpret_cast<const float2*>(sc + kKeys + 8 + 2 * t);
          // (0: a key that is not there)
          auto fits = [](float x) -> bool { return x == 0.0f || (x >= 0x1p-15f && x <= 0x1p7f); };
          const bool small = fits(v0.x) && fits(v0.y) && fits(v1.x) && fits(v1.y);
          if (__all_sync(0xffffffffu, small)) {
            const uint32_t pf[4] = {
                pack2(s[0][0], s[0][1], (__half*)nullptr), pack2(s[0][2], s[0][3], (__half*)nullptr),
                pack2(s[1][0], s[1][1], (__half*)nullptr), pack2(s[1][2], s[1][3], (__half*)nullptr)};
            const uint32_t sv[2] = {pack2(v0.x, v0.y, (__half*)nullptr), pack2(v1.x, v1.y, (__half*)nullptr)};
#pragma unroll
            for (int k = 0; k < KSTEPS; k += 2) {
              uint32_t b[4];
              ldsm_x4_t(b, unit_at(vbase, key_w + (mi & 1) * 8 + mr, k + (mi >> 1)));
#pragma unroll
              for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int odd = 0; odd < 2; ++odd) {
                  const uint32_t c0 = __byte_perm(b[2 * u], 0, odd ? 0x4431 : 0x4420);
                  const uint32_t c1 = __byte_perm(b[2 * u + 1], 0, odd ? 0x4431 : 0x4420);
                  mma16<false>(o[2 * (k + u) + odd], pf, mul_h2(cvt_e4m3x2(c0), sv[0]) & keep[0],
                               mul_h2(cvt_e4m3x2(c1), sv[1]) & keep[1]);
                }
            }
          } else {
            const uint32_t pf[4] = {pack2(s[0][0], s[0][1], (T*)nullptr), pack2(s[0][2], s[0][3], (T*)nullptr),
                                    pack2(s[1][0], s[1][1], (T*)nullptr), pack2(s[1][2], s[1][3], (T*)nullptr)};
#pragma unroll
            for (int k = 0; k < KSTEPS; k += 2) {
              uint32_t b[4];
              ldsm_x4_t(b, unit_at(vbase, key_w + (mi & 1) * 8 + mr, k + (mi >> 1)));
#pragma unroll
              for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int odd = 0; odd < 2; ++odd) {
                  const uint32_t c0 = __byte_perm(b[2 * u], 0, odd ? 0x4431 : 0x4420);
                  const uint32_t c1 = __byte_perm(b[2 * u + 1], 0, odd ? 0x4431 : 0x4420);
                  mma16<FMT == 1>(o[2 * (k + u) + odd], pf, scaled2(cvt_e4m3x2(c0), v0.x, v0.y, (T*)nullptr) & keep[0],
                                  scaled2(cvt_e4m3x2(c1), v1.x, v1.y, (T*)nullptr) & keep[1]);
                }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);

      if (w.j + 1 == w.nt || i + 1 == hi) {
        // ---- the piece ends: join the eight warps, two rows a lane group
        const int64_t unit0 = i - w.j;  // the unit's first tile
        const bool whole = unit0 >= lo && w.j + 1 == w.nt;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
          l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
          if (t == 0) ml[warp * 16 + g + 8 * h] = make_float2(m[h], l[h]);
        }
        sync_consumers();
        float mt[2], lt[2], f[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mt[h] = -INFINITY;
          lt[h] = 0.0f;
#pragma unroll
          for (int x = 0; x < kConsumers; ++x) {
            const float2 y = ml[x * 16 + g + 8 * h];
            if (y.y != 0.0f) mt[h] = fmaxf(mt[h], y.x);
          }
#pragma unroll
          for (int x = 0; x < kConsumers; ++x) {
            const float2 y = ml[x * 16 + g + 8 * h];
            if (y.y != 0.0f) lt[h] += y.y * ex2_approx(y.x - mt[h]);
          }
          f[h] = l[h] == 0.0f ? 0.0f : ex2_approx(m[h] - mt[h]);
        }
        // column of element e of output tile k
        auto col = [&](int k, int e) -> int { return Q8 ? 16 * (k >> 1) + (k & 1) + 4 * t + 2 * e : 8 * k + 2 * t + e; };
        // warps 4-7 hand their rows to warps 0-3, which add theirs: four sums
        float* mine = merge + (warp & 3) * 16 * D;
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
          if ((warp >= 4) == (pass == 0)) {
#pragma unroll
            for (int k = 0; k < OT; ++k)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float* at = mine + merge_at<D>(g + 8 * (e >> 1), col(k, e & 1));
                // a warp that saw no key leaves zeros, whatever 0 * its sums is
                const float x = l[e >> 1] == 0.0f ? 0.0f : o[k][e] * f[e >> 1];
                *at = pass == 0 ? x : *at + x;
              }
          }
          sync_consumers();
        }
        // ---- write out: warp x the rows x and x + 8
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const int r = warp + 8 * h;
          const Row row = row_of(p, w, r);
          float mr2 = -INFINITY, lr = 0.0f;
          for (int x = 0; x < kConsumers; ++x) {
            const float2 y = ml[x * 16 + r];
            if (y.y != 0.0f) mr2 = fmaxf(mr2, y.x);
          }
          for (int x = 0; x < kConsumers; ++x) {
            const float2 y = ml[x * 16 + r];
            if (y.y != 0.0f) lr += y.y * ex2_approx(y.x - mr2);
          }
          bool bad = false;
          for (int d = lane; d < D; d += 32) {
            float* at = merge + merge_at<D>(r, d);
            const float x = (at[0] + at[16 * D]) + (at[32 * D] + at[48 * D]);
            bad = bad || (__float_as_uint(x) & 0x7fffffffu) >= 0x7f800000u;
            at[0] = x;
          }
          bad = __any_sync(0xffffffffu, bad) && row.valid && lr > 0.0f && lr <= 3.4028234663852886e38f;
          const T* q = static_cast<const T*>(p.Q) + int64_t(w.s.q0 + row.token) * p.q_token + row.head * p.q_head;
          const int first = int((whole || unit0 >= lo) ? 0 : lo - unit0) * kKeys;
          if (ok && bad)
            redo_row<T, D, Q8>(p, w.b, w.s.k0, w.hk, q, first, min(row.lim, (w.j + 1) * kKeys), mr2, merge, r);
          __syncwarp();
          if (!ok || !row.valid) continue;
          if (whole) {
            const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
            T* out = static_cast<T*>(p.O) + int64_t(w.s.q0 + row.token) * p.o_token + row.head * p.o_head;
            for (int d = lane; d < D; d += 32) stf(out + d, lr == 0.0f ? 0.0f : merge[merge_at<D>(r, d)] * inv);
          } else {
            // a piece of a unit that began in an earlier block goes to the
            // first place, one that goes on in the next block to the second
            const int64_t at = (c_id * 2 + (unit0 >= lo ? 1 : 0)) * 16 + r;
            if (lane == 0) a.part_ml[at] = make_float2(mr2, lr);
            for (int d = lane; d < D; d += 32) a.part_o[at * D + d] = merge[merge_at<D>(r, d)];
          }
        }
        sync_consumers();
        fresh = true;
      }
      w.step(p);  // a warp that gave up keeps walking: the others meet it where pieces end
    }
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
  int b;
  if (p.cu_q == nullptr) {
    b = t / p.uniform_n;
  } else {
    int lo = 0, hi = p.batch;  // first sequence that begins behind t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.cu_q + mid) <= t) lo = mid + 1; else hi = mid;
    }
    b = lo - 1;
  }
  if (b < 0 || b >= p.batch) return;
  const Seq s = seq_of(p, b);
  if (t < s.q0 || t >= s.q0 + s.n) return;
  const int hk = h / p.group, q = (t - s.q0) * p.group + h - hk * p.group;
  const int nt = unit_tiles(s.len), nrt = row_tiles(s.n, p.group);
  const int64_t total = a.plan[p.batch], used = a.plan[p.batch + 1];
  const int64_t first = a.plan[b] + (int64_t(hk) * nrt + (q >> 4)) * nt;
  // block that holds a tile: the last c with c * total / used <= tile
  const int64_t c0 = min(((first + 1) * used - 1) / total, used - 1);
  const int64_t c1 = min(((first + nt) * used - 1) / total, used - 1);
  if (c0 >= c1) return;  // whole in one block: written there
  auto at = [&](int64_t c) -> int64_t { return (c * 2 + (first_tile(c, total, used) <= first ? 1 : 0)) * 16 + (q & 15); };
  float m = -INFINITY;
  for (int64_t c = c0 + lane; c <= c1; c += 32) {
    const float2 ml = a.part_ml[at(c)];
    if (ml.y != 0.0f) m = fmaxf(m, ml.x);
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
  float l = 0.0f, o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.0f;
  for (int64_t c = c0; c <= c1; ++c) {
    const int64_t x = at(c);
    const float2 ml = a.part_ml[x];
    if (ml.y == 0.0f) continue;
    const float wgt = ex2_approx(ml.x - m);
    l = fmaf(wgt, ml.y, l);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = fmaf(wgt, a.part_o[x * D + lane * N + i], o[i]);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < N; ++i) stf(out + i, l == 0.0f ? 0.0f : o[i] * inv);
}

// ------------------------------------------------------------------ host
int64_t decode_blocks(const DeviceInfo& dev) { return dev.num_sms; }

template <int FMT, int D, bool Q8>
cudaError_t launch_decode_typed(const DecodeParams& a, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t s) {
  using Cfg = DecodeCfg<D, Q8>;
  using T = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
  auto kern = attention_decode_kernel<FMT, D, Q8>;
  static unsigned long long smem_set = 0;
  cudaError_t e = set_smem_once(kern, int(Cfg::SMEM), smem_set);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  apply_pdl(cfg, attr, 0);
  e = cudaLaunchKernelEx(&cfg, kern, tk, tv, a);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(unsigned((int64_t(a.p.tokens_q) * a.p.heads_q + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, attention_decode_combine<T, D>, a);
}

}  // namespace

bool seq_decode_ok(const SeqProblem& p, int dtype, int kv_dtype) {
  return (dtype == CMPX_F16 || dtype == CMPX_BF16) && (p.d == 64 || p.d == 128) && seq_tma_ok(p, kv_dtype) &&
         seq_rows_ok(p.Q, p.q_token, p.tokens_q, 8) && seq_rows_ok(p.Q, p.q_head, p.heads_q, 8) &&
         (int64_t(p.tokens_q) * p.heads_q + 3) / 4 <= 0x7fffffffLL;
}

size_t seq_decode_workspace(const SeqProblem& p, const DeviceInfo& dev) {
  return size_t(decode_blocks(dev)) * 2 * 16 * (size_t(p.d) * 4 + 8) + (size_t(p.batch) + 2) * 8;
}

cudaError_t launch_seq_decode(const SeqProblem& p, int dtype, int kv_dtype, void* ws, const DeviceInfo& dev, int* err,
                              cudaStream_t s) {
  const bool paged = p.table != nullptr, q8 = kv_dtype == CMPX_E4M3;
  DecodeParams a = {};
  a.p = p;
  a.box_rows = paged && p.page_size < kKeys ? p.page_size : kKeys;
  a.blocks = int(decode_blocks(dev));
  a.min_tiles = 1;
  a.part_o = static_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + int64_t(a.blocks) * 2 * 16 * p.d);
  a.plan = reinterpret_cast<int64_t*>(a.part_ml + int64_t(a.blocks) * 2 * 16);
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
