// Attention of a few query rows per sequence over the 8-bit KV cache: decode (one row per query head)
// and short chunks with at most 16 rows per KV head.
//
// Every (sequence, KV head) cache is a run of tiles of 64 positions -- those that hold the first
// visible positions and those from the window's begin to the last row; the runs are laid end to end
// and every CTA takes an equal, contiguous share of that line.  The lengths are read on the device:
// each CTA adds up the runs of the batch (a scan of `batch` integers, about a microsecond) and finds
// its share, so a captured graph follows the lengths.  Six warps:
//   warps 0-3  32 positions of every other tile each: S^T = K Q^T and O^T += V^T P^T as mma.sync
//              m16n8k16 on fp16 -- positions and elements fill the M dimension, the few query rows
//              the N dimension of 8 (up to 16: two of them).  e4m3 converts to fp16 exactly, two codes
//              an instruction, straight from the bytes of the tile: a lane's share of a K row is 32
//              consecutive bytes (the order of the 128 elements in the contraction is free, as long
//              as Q's is the same), and its share of V is 16 consecutive bytes of four rows, whose
//              bytes two permutes pair up.
//   warp 4     TMA producer: K and V tiles (128-byte swizzle) and their exponent bytes, 4 stages of
//              16 KB
//   warp 5     the piece's query rows, as fp16 scaled by a power of two (exact for bf16 and fp16)
// The row exponents never touch the products.  With e_k, e_v those of a position,
//     t = S 2^e_k scale log2(e) + e_v,   P = 2^(t - max t),   O += P c_v,   l += P 2^-e_v
// and O / l is the attention: sums in fp32, P rounded to fp16 (11 bits; it is at most 2^8, since O is
// rescaled only when the running maximum has grown by more than that).
//
// A run that lies in one share is written out; a run that was cut leaves a normalised partial and its
// log-sum-exp per piece, merged by a second, dependent launch in a fixed order.
//
// HBM-bound: 258 bytes per visible position and KV head, read once.  48 sequences of 3000 to 32768 positions, 8 KV
// heads: 278 us in the kernel, 6.4 TB/s; 64 of 300 to 4096: 59 us, 5 TB/s, where fill, drain and short runs show.
#include "q8.cuh"
#include "tc5.cuh"
#include "tma.cuh"

namespace b200attn {

namespace q8d {

using namespace q8;
using namespace tma;

constexpr int kConsumerWarps = 4;
constexpr int kConsumerThreads = kConsumerWarps * 32;
constexpr int kThreads = kConsumerThreads + 64;
constexpr int kStages = 4;
// Tile g of a share lies in stage g % kStages and belongs to consumer pair g % 2.  With an even number of
// stages a pair sees every phase of its stages' barriers; with an odd one it would see every other, and a
// wait on a phase's parity could not tell a phase from the one two before.
static_assert(kStages % 2 == 0, "stages are owned by consumer pairs");
constexpr int kTileN = 64;
constexpr uint32_t kTile = kTileN * 128;             // K or V codes of a tile
constexpr uint32_t kStageBytes = 2 * kTile;
constexpr uint32_t kOffCombine = kStages * kStageBytes;              // [4 warps][8 rows][128] fp32
constexpr uint32_t kOffExp = kOffCombine + kConsumerWarps * 8 * 512; // [stage][K, V][64]
constexpr uint32_t kOffQ = kOffExp + kStages * 128;                  // [16][128] fp16
constexpr uint32_t kOffQs = kOffQ + 16 * 256;                        // [16] fp32: what a row's scores are multiplied by
constexpr uint32_t kOffMl = kOffQs + 64;                             // [4][16][max, sum]
constexpr uint32_t kOffScan = kOffMl + kConsumerWarps * 16 * 8;      // scan scratch: 8 + 4 ints
constexpr uint32_t kOffBar = kOffScan + 64;
constexpr uint32_t kSmemTotal = kOffBar + 128;
static_assert(kSmemTotal <= 115712, "two CTAs per SM");
constexpr int kMaxCtas = 296;                        // two per SM
constexpr int kPieceCost = 4;                        // what a run costs besides its tiles, in tiles
constexpr float kLazy = 8.0f;                        // log2 of how far P may exceed 1 before O is rescaled

enum { BAR_FULL = 0, BAR_EMPTY = kStages, BAR_QREADY = 2 * kStages, BAR_QFREE, BAR_COUNT };
static_assert(BAR_COUNT * 8 + 8 <= 128, "barrier block");

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumerThreads) : "memory"); }

using Seq = Span<kTileN>;

__device__ __forceinline__ Seq seq_of(const Q8AttnParams &p, int b) {
  Seq s;
  int limit = min(p.max_kv_len, p.c.max_pos);
  if (p.kv_len) {
    const int len = __ldg(p.kv_len + b);
    if (len > limit) report(p.c.error_flag, kStatusLengthBeyondBound);
    s.t0 = b;
    s.nq = 1;
    s.pos0 = min(len, limit) - 1;
  } else {
    chunk_rows(p, b, true, s.t0, s.nq, s.pos0, limit);
    s.nq = min(s.nq, p.max_new);
  }
  s.cover(p, limit);
  return s;
}

// The pieces of one CTA's share, in order.
struct Walk {
  int b, kvh, i0, i1;
  long left;
  Seq s;
  // `offset`: the share's begin on the runs of sequence b; a run is kPieceCost, then its tiles.  False: the
  // share is all cost and no tile.
  __device__ __forceinline__ bool begin(const Q8AttnParams &p, int b_, long offset, long share) {
    b = b_;
    s = seq_of(p, b);
    const int one = s.n_tiles + kPieceCost;
    kvh = static_cast<int>(offset / one);
    const int at = static_cast<int>(offset - static_cast<long>(kvh) * one);
    i0 = max(0, at - kPieceCost);
    left = share - max(0, kPieceCost - at);
    i1 = static_cast<int>(min(static_cast<long>(s.n_tiles), i0 + left));
    return left > 0;
  }
  __device__ __forceinline__ bool next(const Q8AttnParams &p) { // false: the share is done
    left -= i1 - i0 + kPieceCost;
    if (left <= 0) return false;
    if (++kvh == p.c.n_kv_heads) {
      kvh = 0;
      do {
        if (++b >= p.c.batch) return false;
        s = seq_of(p, b);
      } while (s.n_tiles == 0);
    }
    i0 = 0;
    i1 = static_cast<int>(min(static_cast<long>(s.n_tiles), left));
    return true;
  }
};
__device__ __forceinline__ int run_cost(const Seq &s) { return s.n_tiles > 0 ? s.n_tiles + kPieceCost : 0; }

// A piece's partial goes to slot 2 c (the share's first piece) or 2 c + 1 (its last one).  Which slots
// a cut run left: first and last CTA, and the slot of the first; of the others it is 2 c.
struct RunInfo {
  int c0, c1, slot0, pad;
};

struct Ws {
  float *o, *lse; // [slot][rows][128], [slot][rows]
  RunInfo *info;  // [batch * kv heads]
};

} // namespace q8d

struct Q8DecodeParams {
  Q8AttnParams a;
  q8d::Ws ws;
  int rows;       // rows of a partial: max_new * group
};

template <typename T, int NH> // NH: query rows in eights
__global__ void __launch_bounds__(q8d::kThreads, 2)
attn_q8_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ CUtensorMap map_k16, const __grid_constant__ CUtensorMap map_v16, const Q8DecodeParams dp) {
  using namespace q8d;
  const Q8AttnParams &p = dp.a;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t smem_base = smem_u32(smem);
  int *scan = reinterpret_cast<int *>(smem + kOffScan);
  float *red_ml = reinterpret_cast<float *>(smem + kOffMl);
  volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + kOffBar + BAR_COUNT * 8);
  auto bar = [&](int i) { return smem_base + kOffBar + 8u * i; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = p.group, kvH = p.c.n_kv_heads;

  cudaTriggerProgrammaticLaunchCompletion();
  if (tid == 0) {
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(BAR_FULL + s), 1);
      mbar_init(bar(BAR_EMPTY + s), 2);
    }
    mbar_init(bar(BAR_QREADY), 1);
    mbar_init(bar(BAR_QFREE), kConsumerWarps);
    *abort_flag = 0;
    fence_barrier_init();
  }
  cudaGridDependencySynchronize(); // lengths, rows, cache and scratch may be the preceding kernels'

  // ---- this CTA's share: tiles of the whole batch, and the sequence its first tile belongs to
  const int per = (p.c.batch + kThreads - 1) / kThreads;
  const int b_lo = min(p.c.batch, tid * per), b_hi = min(p.c.batch, b_lo + per);
  int mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += run_cost(seq_of(p, b));
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) scan[warp] = incl;
  if ((smem_base & 1023u) != 0 && tid == 0) report(p.c.error_flag, 30);
  __syncthreads();
  if ((smem_base & 1023u) != 0) return;
  int before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  const long W = static_cast<long>(total) * kvH;
  const int n = static_cast<int>(min(static_cast<long>(gridDim.x), W));
  const int c = blockIdx.x;
  if (c >= n) return;
  const long x0 = share_begin(W, n, c), x1 = share_begin(W, n, c + 1);
  if (x0 >= static_cast<long>(before) * kvH && x0 < static_cast<long>(before + mine) * kvH) {
    long at = static_cast<long>(before) * kvH;
    for (int b = b_lo; b < b_hi; ++b) {
      const long run = static_cast<long>(run_cost(seq_of(p, b))) * kvH;
      if (x0 < at + run) {
        scan[8] = b;
        scan[9] = static_cast<int>(x0 - at);
        break;
      }
      at += run;
    }
  }
  __syncthreads();
  const int b_first = scan[8], off_first = scan[9];

  if (warp == kConsumerWarps) {
    // ------------------------------------------------------------------ TMA producer
    Walk w;
    if (!w.begin(p, b_first, off_first, x1 - x0)) return;
    uint32_t g = 0;
    do {
      for (int base = w.i0; base < w.i1; base += 32) {
        // the lanes look up the pages of 32 tiles at once
        const int mine_i = base + lane;
        int outer = w.b, row = 0;
        if (mine_i < w.i1) {
          row = w.s.tile(mine_i) * kTileN;
          if (p.c.pg.table) {
            outer = __ldg(p.c.pg.table + static_cast<long>(w.b) * p.c.pg.table_stride + (row >> p.c.pg.page_shift));
            row &= (1 << p.c.pg.page_shift) - 1;
            if (static_cast<unsigned>(outer) >= static_cast<unsigned>(p.c.pg.n_pages)) {
              report(p.c.error_flag, kStatusOutsideCache);
              outer = 0;
            }
          }
        }
        const int cnt = min(32, w.i1 - base);
        for (int k = 0; k < cnt; ++k, ++g) {
          const int outer_k = __shfl_sync(0xffffffffu, outer, k), row_k = __shfl_sync(0xffffffffu, row, k);
          const int s = g % kStages;
          bool ok = true;
          if (lane == 0) {
            ok = mbar_wait(bar(BAR_EMPTY + s), ((g / kStages) & 1) ^ 1, abort_flag, p.c.error_flag, 31);
            if (ok) {
              // rows of the tile that some query row sees, in groups of 16
              const int tpos = w.s.tile(base + k) * kTileN;
              const int r0 = (tpos < w.s.ns ? 0 : max(0, w.s.lo - tpos)) & ~15;
              const int r1 = (min(kTileN, w.s.end - tpos) + 15) & ~15;
              const uint32_t full = bar(BAR_FULL + s);
              const uint32_t dk = smem_base + s * kStageBytes, dv = dk + kTile;
              const uint32_t dx = smem_base + kOffExp + s * 128;
              const uint32_t rows = static_cast<uint32_t>(r1 - r0);
              mbar_expect_tx(full, rows * 258);
              if (rows == kTileN) {
                tma_load_4d(dk, &map_k, full, 0, row_k, w.kvh, outer_k);
                tma_load_4d(dv, &map_v, full, 0, row_k, w.kvh, outer_k);
              } else {
                for (int r = r0; r < r1; r += 16) {
                  tma_load_4d(dk + r * 128, &map_k16, full, 0, row_k + r, w.kvh, outer_k);
                  tma_load_4d(dv + r * 128, &map_v16, full, 0, row_k + r, w.kvh, outer_k);
                }
              }
              const long xo = static_cast<long>(outer_k) * p.c.x_outer + w.kvh * p.c.x_head + row_k + r0;
              bulk_load(dx + r0, p.c.kx + xo, rows, full);
              bulk_load(dx + 64 + r0, p.c.vx + xo, rows, full);
            }
          }
          if (!__shfl_sync(0xffffffffu, static_cast<int>(ok), 0)) return;
        }
      }
    } while (w.next(p));
    return;
  }

  if (warp == kConsumerWarps + 1) {
    // ------------------------------------------------------------------ query rows
    Walk w;
    if (!w.begin(p, b_first, off_first, x1 - x0)) return;
    unsigned char *q_s = smem + kOffQ;
    float *qs = reinterpret_cast<float *>(smem + kOffQs);
    int it = 0;
    do {
      const bool wait_ok = it == 0 || mbar_wait(bar(BAR_QFREE), (it - 1) & 1, abort_flag, p.c.error_flag, 32);
      if (!__all_sync(0xffffffffu, wait_ok)) return;
      const int nrows = w.s.nq * G;
#pragma unroll
      for (int it4 = 0; it4 < 2 * NH; ++it4) {
        const int rho = it4 * 4 + (lane >> 3), j = lane & 7; // eight lanes per row, 16 elements each
        uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
        if (rho < nrows) {
          const int tok = rho / G;
          const T *src = static_cast<const T *>(p.q) + static_cast<long>(w.s.t0 + tok) * p.q_row + (w.kvh * G + rho - tok * G) * kHeadDim + 16 * j;
          u0 = *reinterpret_cast<const uint4 *>(src);
          u1 = *reinterpret_cast<const uint4 *>(src + 8);
        }
        float f[16];
        const uint32_t ww[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 v = Elem<T>::unpack(ww[e]);
          f[2 * e] = v.x, f[2 * e + 1] = v.y;
          top = max(top, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // the row's largest magnitude to 2^13 .. 2^14: an element keeps all its bits down to 2^-29 of it
        int e = max(static_cast<int>(top >> 23) - 127, -100);
        if (top >= 0x7f800000u) e = 13; // not finite: as it is
        const float up = pow2i(13 - e);
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = Elem<__half>::pack(f[2 * i] * up, f[2 * i + 1] * up);
        uint4 *dst = reinterpret_cast<uint4 *>(q_s + rho * 256 + j * 32);
        dst[0] = make_uint4(h[0], h[1], h[2], h[3]);
        dst[1] = make_uint4(h[4], h[5], h[6], h[7]);
        if (j == 0) qs[rho] = p.scale_log2 * pow2i(e - 13);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(BAR_QREADY));
      ++it;
    } while (w.next(p));
    return;
  }

  // -------------------------------------------------------------------- consumers
  // Fragments: rows of K are the M dimension, query rows (8 per NH) the N dimension, so that few query
  // rows cost few products and accumulators.  This lane: positions g0 and g0 + 8 of a group of 16,
  // query rows 2 cq and 2 cq + 1 of S; elements 16 g0 + x of O for the same query rows.
  const int g0 = lane >> 2, cq = lane & 3;
  const float kNegInf = -INFINITY, kNan = __int_as_float(0x7fc00000);
  Walk w;
  if (!w.begin(p, b_first, off_first, x1 - x0)) return;
  uint32_t g = 0;
  int it = 0;
  bool ok = true; // a wait that gave up leaves a status; the warp goes on to the end without its tiles
  do {
    ok = ok && mbar_wait(bar(BAR_QREADY), it & 1, abort_flag, p.c.error_flag, 33);
    // contraction order: k-step ks of this lane covers elements 32 cq + 4 ks + {0, 1} and + {2, 3}
    uint32_t qb[NH][8][2];
    float qs[NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
      const uint4 *r = reinterpret_cast<const uint4 *>(smem + kOffQ + (8 * nh + g0) * 256 + cq * 64);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint4 v = r[x];
        qb[nh][2 * x][0] = v.x, qb[nh][2 * x][1] = v.y, qb[nh][2 * x + 1][0] = v.z, qb[nh][2 * x + 1][1] = v.w;
      }
      const float2 s2 = *reinterpret_cast<const float2 *>(smem + kOffQs + (8 * nh + 2 * cq) * 4);
      qs[nh][0] = s2.x, qs[nh][1] = s2.y;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(BAR_QFREE));

    const int nrows = w.s.nq * G;
    // every row sees all of what ends before the first row's position and begins at or behind the last
    // row's window, or lies among the first positions
    const int all_end = min(w.s.pos0 + 1, w.s.end), all_lo = window_begin(w.s.pos0 + w.s.nq - 1, p.window);

    float o[NH][8][4];
    float m[NH][2], l[NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
      for (int x = 0; x < 8; ++x) o[nh][x][0] = o[nh][x][1] = o[nh][x][2] = o[nh][x][3] = 0.f;
      m[nh][0] = m[nh][1] = kNegInf;
      l[nh][0] = l[nh][1] = 0.f;
    }

    // a tile is the work of two warps, 32 positions (two groups of 16) each; the other two have the next
    for (int i = w.i0; i < w.i1; ++i, ++g) {
      if ((g & 1) != static_cast<uint32_t>(warp >> 1)) continue;
      const int s = g % kStages;
      const int row0 = (warp & 1) * 32, col0 = w.s.tile(i) * kTileN + row0;
      const bool some = col0 < w.s.end && (col0 + 31 >= w.s.lo || col0 < w.s.ns);
      const bool all = col0 + 32 <= all_end && (col0 >= all_lo || col0 + 32 <= p.n_sink);
      ok = ok && mbar_wait(bar(BAR_FULL + s), (g / kStages) & 1, abort_flag, p.c.error_flag, 34);
      if (__all_sync(0xffffffffu, ok) && some) {
        const uint32_t st_k = smem_base + s * kStageBytes + row0 * 128, st_v = st_k + kTile;
        const unsigned char *ex = smem + kOffExp + s * 128 + row0;
        float sc[2][NH][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t kw[2][8];
#pragma unroll
          for (int rr = 0; rr < 2; ++rr)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              lds128(kw[rr] + 4 * x, st_k + (16 * u + 8 * rr + g0) * 128 + (((2 * cq + x) ^ g0) << 4));
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) sc[u][nh][0] = sc[u][nh][1] = sc[u][nh][2] = sc[u][nh][3] = 0.f;
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            uint32_t ka[4];
            cvt_e4m3x4_f16x4(kw[0][ks], ka[0], ka[2]);
            cvt_e4m3x4_f16x4(kw[1][ks], ka[1], ka[3]);
#pragma unroll
            for (int nh = 0; nh < NH; ++nh) mma_16816<__half>(sc[u][nh], ka, qb[nh][ks][0], qb[nh][ks][1]);
          }
        }
        // V: 16 bytes (elements 16 g0 ..) of rows 2 cq + {0, 1, 8, 9} of either group
        uint32_t vw[2][4][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int r = 2 * cq + (x & 1) + (x >> 1) * 8;
            lds128(vw[u][x], st_v + (16 * u + r) * 128 + ((g0 ^ (r & 7)) << 4));
          }
        // t = S 2^e_k scale + e_v; exponents of this lane's four positions
        float vinv[2][2], top[NH][2];
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) top[nh][0] = top[nh][1] = kNegInf;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int rr = 0; rr < 2; ++rr) {
            const uint32_t kx = ex[16 * u + 8 * rr + g0], vx = ex[64 + 16 * u + 8 * rr + g0];
            const float kf = (kx == kPoison || vx == kPoison) ? kNan : __uint_as_float(kx << 23);
            const float ev = static_cast<float>(static_cast<int>(vx) - 127);
            vinv[u][rr] = __uint_as_float((254u - min(vx, 253u)) << 23);
#pragma unroll
            for (int nh = 0; nh < NH; ++nh)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float &t = sc[u][nh][2 * rr + e];
                t = fmaf(t, qs[nh][e] * kf, ev);
                if (!all) {
                  const int j = col0 + 16 * u + 8 * rr + g0, pr = w.s.pos0 + (8 * nh + 2 * cq + e) / G;
                  if (!(j < min(pr + 1, w.s.end) && (j >= window_begin(pr, p.window) || j < p.n_sink))) t = kNegInf;
                }
                top[nh][e] = fmaxf(top[nh][e], t);
              }
          }
        bool grow = false;
#pragma unroll
        for (int nh = 0; nh < NH; ++nh)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top[nh][e] = fmaxf(top[nh][e], __shfl_xor_sync(0xffffffffu, top[nh][e], d));
            grow |= top[nh][e] > m[nh][e] + kLazy;
          }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int nh = 0; nh < NH; ++nh)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const bool up = top[nh][e] > m[nh][e] + kLazy;
              const float f = up ? tc5::ex2(m[nh][e] - top[nh][e]) : 1.f;
              if (up) m[nh][e] = top[nh][e];
              l[nh][e] *= f;
#pragma unroll
              for (int x = 0; x < 8; ++x) o[nh][x][e] *= f, o[nh][x][2 + e] *= f;
            }
        }
        // P, its 8 x 8 blocks turned so that a lane holds two positions of query row g0
        uint32_t pb[2][NH][2];
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
          const float ms0 = m[nh][0] == kNegInf ? 0.f : m[nh][0], ms1 = m[nh][1] == kNegInf ? 0.f : m[nh][1]; // nothing seen yet: P = 0
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
              const float p0 = tc5::ex2(sc[u][nh][2 * rr] - ms0), p1 = tc5::ex2(sc[u][nh][2 * rr + 1] - ms1);
              l[nh][0] = fmaf(p0, vinv[u][rr], l[nh][0]);
              l[nh][1] = fmaf(p1, vinv[u][rr], l[nh][1]);
              pb[u][nh][rr] = transpose8x8(Elem<__half>::pack(p0, p1));
            }
        }
        if (!all) {
          // a row nobody sees may hold anything: a zero weight must not meet a NaN code
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int j = col0 + 16 * u + 2 * cq + (x & 1) + (x >> 1) * 8;
              if (!(j < w.s.end && (j >= w.s.lo || j < w.s.ns))) vw[u][x][0] = vw[u][x][1] = vw[u][x][2] = vw[u][x][3] = 0u;
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const uint32_t lo2 = __byte_perm(vw[u][0][q4], vw[u][1][q4], hh ? 0x7362 : 0x5140);
              const uint32_t hi2 = __byte_perm(vw[u][2][q4], vw[u][3][q4], hh ? 0x7362 : 0x5140);
              uint32_t va[4];
              cvt_e4m3x4_f16x4(lo2, va[0], va[1]);
              cvt_e4m3x4_f16x4(hi2, va[2], va[3]);
#pragma unroll
              for (int nh = 0; nh < NH; ++nh) mma_16816<__half>(o[nh][2 * q4 + hh], va, pb[u][nh][0], pb[u][nh][1]);
            }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(BAR_EMPTY + s));
    }

    // ---- the four warps' states of the piece -> its result.  Accumulator x of a lane holds elements
    //      16 g0 + 2 x and 16 g0 + 2 x + 1 of its two query rows.
#pragma unroll
    for (int nh = 0; nh < NH; ++nh)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nh][e] += __shfl_xor_sync(0xffffffffu, l[nh][e], d);
        if (g0 == 0) *reinterpret_cast<float2 *>(red_ml + (warp * 16 + 8 * nh + 2 * cq + e) * 2) = make_float2(m[nh][e], l[nh][e]);
      }
    consumer_sync();
    auto row_ml = [&](int row, float &M, float &L) {
      M = kNegInf;
#pragma unroll
      for (int x = 0; x < kConsumerWarps; ++x) M = fmaxf(M, red_ml[(x * 16 + row) * 2]);
      const float ms = M == kNegInf ? 0.f : M;
      L = 0.f;
#pragma unroll
      for (int x = 0; x < kConsumerWarps; ++x) L += exp2f(red_ml[(x * 16 + row) * 2] - ms) * red_ml[(x * 16 + row) * 2 + 1];
    };
    const bool whole = w.i0 == 0 && w.i1 == w.s.n_tiles;
    const int slot = 2 * c + (it == 0 ? 0 : 1);
    float *buf = reinterpret_cast<float *>(smem + kOffCombine);
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
      if (nh * 8 < nrows) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float M, L;
          row_ml(8 * nh + 2 * cq + e, M, L);
          // L is NaN where a poisoned row was seen, and 0 where nothing was
          const float f = L == 0.f ? 0.f : exp2f(m[nh][e] - (M == kNegInf ? 0.f : M)) / L;
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            // four elements 16 g0 + 4 q4, their place turned by the row so that eight lanes hit eight banks
            const float4 v = make_float4(o[nh][2 * q4][e] * f, o[nh][2 * q4][2 + e] * f, o[nh][2 * q4 + 1][e] * f, o[nh][2 * q4 + 1][2 + e] * f);
            reinterpret_cast<float4 *>(buf)[(warp * 8 + 2 * cq + e) * 32 + ((4 * g0 + q4) ^ cq)] = v;
          }
        }
      }
      consumer_sync();
      const int rr = tid >> 4, rho = rr + 8 * nh;
      if (rho < nrows) {
        const int tok = rho / G;
        const long t = w.s.t0 + tok;
        const int h = w.kvh * G + rho - tok * G;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int ch = (tid & 15) + 16 * k;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int x = 0; x < kConsumerWarps; ++x) {
            const float4 u = reinterpret_cast<const float4 *>(buf)[(x * 8 + rr) * 32 + (ch ^ (rr >> 1))];
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
          }
          if (whole) {
            uint2 u;
            u.x = Elem<T>::pack(v.x, v.y);
            u.y = Elem<T>::pack(v.z, v.w);
            *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + t * p.out_row + h * kHeadDim + 4 * ch) = u;
          } else {
            *reinterpret_cast<float4 *>(dp.ws.o + (static_cast<long>(slot) * dp.rows + rho) * kHeadDim + 4 * ch) = v;
          }
        }
        if (!whole && (tid & 15) == 0) {
          float M, L;
          row_ml(rho, M, L);
          dp.ws.lse[static_cast<long>(slot) * dp.rows + rho] = L == 0.f ? kNegInf : (M == kNegInf ? 0.f : M) + log2f(L);
        }
      }
      consumer_sync(); // the buffer and red_ml may be written again
    }
    if (w.i0 == 0 && tid == 0) {
      // this CTA holds the run's first tile: it says which CTAs hold the others
      const long first = x1 - w.left; // the first tile's place on the line
      const int last = share_of(W, n, first + w.s.n_tiles - 1);
      RunInfo r;
      r.c0 = c, r.c1 = last, r.slot0 = slot, r.pad = 0;
      dp.ws.info[static_cast<long>(w.b) * kvH + w.kvh] = r;
    }
    ++it;
  } while (w.next(p));
}

// Merges the pieces of the runs that were cut, and zeroes the rows that see nothing.
template <typename T> __global__ void __launch_bounds__(32 * kMergeWarps) attn_q8_merge_kernel(const Q8DecodeParams dp, int split) {
  using namespace q8d;
  const Q8AttnParams &p = dp.a;
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
  const int kvH = p.c.n_kv_heads, G = p.group;
  const int b = blockIdx.x / kvH, kvh = blockIdx.x - b * kvH;
  const RunInfo info = dp.ws.info[blockIdx.x]; // of a run without tiles: whatever was there, not used
  const Seq s = seq_of(p, b);
  if (s.n_tiles > 0 && info.c1 <= info.c0) return; // the run was not cut
  merge_rows(dp.ws.o, dp.ws.lse, s.n_tiles > 0 ? info.c1 - info.c0 + 1 : 0, s.nq * G, split,
             [&](int i, int rho) { return static_cast<long>(i == 0 ? info.slot0 : 2 * (info.c0 + i)) * dp.rows + rho; },
             [&](int rho, const float4 &v) {
               const int tok = rho / G;
               uint2 u;
               u.x = Elem<T>::pack(v.x, v.y);
               u.y = Elem<T>::pack(v.z, v.w);
               *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + static_cast<long>(s.t0 + tok) * p.out_row +
                                          (kvh * G + rho - tok * G) * kHeadDim + (threadIdx.x & 31) * 4) = u;
             });
}

namespace {

// the shared-memory opt-in is a property of (function, device): set on the first launch per device
template <typename T, int NH> cudaError_t opt_in() {
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !done[dev]) {
    e = cudaFuncSetAttribute(attn_q8_decode_kernel<T, NH>, cudaFuncAttributeMaxDynamicSharedMemorySize, q8d::kSmemTotal);
    if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  }
  return e;
}

template <typename T, int NH>
cudaError_t launch_typed(const Q8DecodeParams &dp, int n_ctas, const CUtensorMap *m, cudaStream_t stream, int *launches) {
  cudaError_t e = opt_in<T, NH>();
  if (e != cudaSuccess) return e;
  e = launch_dependent(attn_q8_decode_kernel<T, NH>, dim3(n_ctas), q8d::kThreads, q8d::kSmemTotal, stream, m[0], m[1], m[2], m[3], dp);
  if (e != cudaSuccess) return e;
  *launches = 1;
  dim3 grid;
  int split;
  merge_shape(static_cast<long>(dp.a.c.batch) * dp.a.c.n_kv_heads, dp.rows, n_ctas, &grid, &split);
  e = launch_dependent(attn_q8_merge_kernel<T>, grid, 32 * kMergeWarps, 0, stream, dp, split);
  if (e != cudaSuccess) return e;
  *launches = 2;
  return cudaGetLastError();
}

int cta_count(int batch, int n_kv_heads, int max_kv_len) {
  const long tiles = static_cast<long>(batch) * n_kv_heads * ((static_cast<long>(max_kv_len) + q8d::kTileN - 1) / q8d::kTileN);
  return static_cast<int>(tiles < q8d::kMaxCtas ? tiles : q8d::kMaxCtas);
}

} // namespace

size_t attn_q8_decode_ws_bytes(int batch, int n_kv_heads, int rows, int max_kv_len) {
  const size_t slots = 2 * static_cast<size_t>(cta_count(batch, n_kv_heads, max_kv_len));
  const size_t parts = (slots * rows * (kHeadDim + 1) * sizeof(float) + 15) / 16 * 16;
  return parts + static_cast<size_t>(batch) * n_kv_heads * sizeof(q8d::RunInfo);
}

cudaError_t launch_attn_q8_decode(const Q8AttnParams &p, bool bf16, cudaStream_t stream, int *launches) {
  *launches = 0;
  const Q8Cache &c = p.c;
  Q8DecodeParams dp{};
  dp.a = p;
  dp.rows = p.max_new * p.group;
  const int n_ctas = cta_count(c.batch, c.n_kv_heads, p.max_kv_len);
  const size_t slots = 2 * static_cast<size_t>(n_ctas);
  dp.ws.o = static_cast<float *>(p.ws);
  dp.ws.lse = dp.ws.o + slots * dp.rows * kHeadDim;
  dp.ws.info = reinterpret_cast<q8d::RunInfo *>(static_cast<char *>(p.ws) + (slots * dp.rows * (kHeadDim + 1) * sizeof(float) + 15) / 16 * 16);
  // (d, position, kv head, sequence), or (d, position in page, kv head, page)
  const uint64_t rows = c.pg.table ? 1ull << c.pg.page_shift : static_cast<uint64_t>(c.max_pos);
  const uint64_t outers = c.pg.table ? static_cast<uint64_t>(c.pg.n_pages) : static_cast<uint64_t>(c.batch);
  CUtensorMap m[4];
  const void *base[2] = {c.k, c.v};
  for (int i = 0; i < 4; ++i)
    if (!make_tensor_map_u8(&m[i], true, base[i & 1], rows, c.n_kv_heads, outers, c.c_pos, c.c_head, c.c_outer, i < 2 ? 64 : 16))
      return cudaErrorNotSupported;
  const bool wide = dp.rows > 8;
  if (bf16)
    return wide ? launch_typed<__nv_bfloat16, 2>(dp, n_ctas, m, stream, launches) : launch_typed<__nv_bfloat16, 1>(dp, n_ctas, m, stream, launches);
  return wide ? launch_typed<__half, 2>(dp, n_ctas, m, stream, launches) : launch_typed<__half, 1>(dp, n_ctas, m, stream, launches);
}

} // namespace b200attn
