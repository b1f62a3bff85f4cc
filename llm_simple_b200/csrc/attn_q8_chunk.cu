// Causal attention of ragged chunks of new tokens over the 8-bit KV cache, on the 5th-generation
// tensor cores.
//
// A block is up to 2 x 128 query rows of one KV head and one sequence: 128 / group tokens times the
// group's heads in each of two tiles A and B, so that every cache tile, once in shared memory, serves
// all heads that share it.  A block walks the tiles of 128 positions that its rows see.  The walks of
// all blocks are laid end to end and every CTA (one per SM) takes an equal, contiguous share of that
// line; where the line is cut inside a block, the pieces leave normalised partials and log-sum-exps
// that a second, dependent launch merges in a fixed order.  The lengths are read on the device.
//
// 16 warps in four groups:
//   warp 0       TMA producer: e4m3 tiles of K and V in boxes of 64 positions, with their exponents
//   warps 1, 2   MMA issuers of A and B: S_X = Q_X K^T, then O_X += P_X V with P from tensor memory
//   warps 4-11   softmax of tile A (4-7) and B (8-11), one thread per query row; they also bring the
//                rows of Q in and the results out
//   warps 12-15  converters: e4m3 -> fp16 operand tiles
// All products run on fp16.  e4m3 codes are exact in it, and Q is scaled by a power of two per row.
// The row exponents of a tile are taken relative to the largest one of the tile, r = max e: the
// converters scale row j by 2^(7 + e_j - r), which is exact for all codes as long as e_j is within 22
// of r (a row 2^22 below its tile's largest loses bits that lie 2^-41 below that row).  Then
//     t = S 2^(r_k - 7) scale log2(e) + (r_v - 7),  P = 2^(t - max t),  O += P V',  l += 2^(7 - r_v) sum P
// where r_k, r_v are constants of the tile: the softmax costs what it costs over 16-bit caches.
// P is rounded to fp16 (at most 2^8: O is rescaled only when the maximum grew by more than that).
// A position outside every row's view is converted to zeros whatever its bytes are; a position whose
// exponent says "not finite" becomes a NaN row of K' and zeros in V', so that exactly the rows that
// see it turn NaN.
//
// A tile is taken in two steps of 64 positions: the softmax warps copy a step's scores to registers and
// free them at once, so that the next step's Q K^T runs while they work.  Tensor memory: S_A, S_B 64
// columns each, P_A, P_B two halves of 32, O_A, O_B 128.
//
// A tile of 128 positions against 256 rows is 2048 cycles of products (63 cycles for 128 x 128 x 16, about
// 50 for the 128 x 64 x 16 of Q K^T, which shared memory feeds) and 2048 of exponentials (16 a cycle).
// Measured 4900: 4096 tokens behind 12288, 40 / 8 heads, 1450 us (830 TFLOP/s).  What bounds it is the
// softmax warps: two on a scheduler, an instruction of each every four to five cycles; without the products
// they take 1270 us, the products and barriers alone 925, the converters 940.
#include "q8.cuh"
#include "tc5.cuh"
#include "tma.cuh"

namespace b200attn {

namespace q8c {

using namespace q8;
using namespace tma;
using namespace tc5;

constexpr int kThreads = 512;
constexpr int kBN = 128;
constexpr uint32_t kHalfTile = 128 * 128;            // [128 rows][64 fp16], swizzled
constexpr uint32_t kTileBytes = 2 * kHalfTile;
constexpr uint32_t kRawBytes = 128 * 128;            // e4m3 tile
constexpr uint32_t kSmemQ = 0;                       // Q_A, Q_B
constexpr uint32_t kSmemK = kSmemQ + 2 * kTileBytes; // two stages
constexpr uint32_t kSmemV = kSmemK + 2 * kTileBytes;
constexpr uint32_t kSmemRaw = kSmemV + 2 * kTileBytes; // K, V
constexpr uint32_t kSmemExp = kSmemRaw + 2 * kRawBytes; // K [128], V [128]
constexpr uint32_t kSmemRef = kSmemExp + 256;        // [4][r_k, r_v]
constexpr uint32_t kSmemScan = kSmemRef + 32;        // 16 + 8 ints
constexpr uint32_t kSmemBar = kSmemScan + 96;
constexpr uint32_t kSmemWalk = kSmemBar + 320;       // [16 warps]
constexpr uint32_t kWalkBytes = 128;
constexpr uint32_t kSmemTotal = kSmemWalk + 16 * kWalkBytes;
static_assert(kSmemTotal <= 232448, "shared memory of one CTA");
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 256; // S_X: 64 columns at kColS + 64 X; P_X: two halves of 32 at kColP + 64 X; O_X
constexpr float kLazy = 8.0f;
constexpr int kMaxCtas = 148;
constexpr int kPieceCost = 6;                        // what a block costs besides its tiles, in tiles: its rows of Q, fill and drain, results.
                                                     // Prompts of 33 to 1024 tokens: 520 us with 0, 359 with 2, 312 with 4, 309 with 8
static_assert((kChunkMaxBatch + 1) * 4 <= 2 * 2 * 128 * 128 * 2, "prefix sums");
// kChunkMaxBatch:                     // prefix sums of the batch lie in the Q tiles while a CTA finds its share

enum { BAR_RAWFULL = 0, BAR_RAWEMPTY = 2, BAR_KFULL = 4, BAR_KEMPTY = 6, BAR_VFULL = 8, BAR_VEMPTY = 10, BAR_QFULL = 12, BAR_QTAKEN = 14,
       BAR_SFULL = 16, BAR_SFREE = 18, BAR_PFULL = 20 /* [half][x] */, BAR_ODONE = 24 /* [half][x] */, BAR_REF = 28, BAR_COUNT = 32 };
static_assert(BAR_COUNT * 8 + 8 <= 320, "barrier block");

using Block = Span<kBN>;

struct Head { // 16 bytes, at the front of the workspace
  int n_blocks, pad[3];
};
// What a block's pieces left: the CTAs c0 .. c1 (c1 < c0: no row sees anything), the slot of the first
// (of the others it is 2 c), and the block's rows.
struct RunInfo {
  int c0, c1, slot0, t0, nq, pad[3];
};

} // namespace q8c

struct Q8ChunkParams {
  Q8AttnParams a;
  int tile_tokens;      // tokens per tile of 128 rows: 128 / group
  q8c::Head *head;
  q8c::RunInfo *info;   // [blocks][kv heads]
  float *o, *lse;       // [slot][2 * tile_tokens * group][128], and without the 128
};

namespace q8c {

// Block blk of sequence b.
__device__ __forceinline__ Block block_of(const Q8ChunkParams &cp, int b, int blk) {
  const Q8AttnParams &p = cp.a;
  int t0, nq, pos0, limit;
  chunk_rows(p, b, false, t0, nq, pos0, limit);
  const int first = blk * 2 * cp.tile_tokens;
  Block s;
  s.t0 = t0 + first;
  s.nq = min(2 * cp.tile_tokens, nq - first);
  s.pos0 = pos0 + first;
  s.cover(p, limit);
  return s;
}
__device__ __forceinline__ int blocks_of(const Q8ChunkParams &cp, int b) {
  int t0, nq, pos0, limit;
  chunk_rows(cp.a, b, blockIdx.x == 0, t0, nq, pos0, limit);
  return (nq + 2 * cp.tile_tokens - 1) / (2 * cp.tile_tokens);
}

// The rows of tile X of a block: their positions, and which tiles of the walk they see.
struct Half {
  int first, n_tok;          // position of the first row; number of tokens (0: the tile is empty)
  int fx, ex;                // besides the tiles of the first positions, tiles [fx, ex) of the walk hold something some row sees
  int ga, gb;                // tiles [ga, gb), and the first `gs` ones: every row sees all of them
  int gs;
  __device__ __forceinline__ void of(const Q8ChunkParams &cp, const Block &s, int x) {
    n_tok = max(0, min(cp.tile_tokens, s.nq - x * cp.tile_tokens));
    first = s.pos0 + x * cp.tile_tokens;
    const int last = min(first + n_tok, s.end) - 1;
    const int skip = s.w0 - s.ns_tiles;  // walk index i >= ns_tiles is cache tile i + skip
    fx = max(s.ns_tiles, window_begin(first, cp.a.window) / kBN - skip);
    ex = n_tok > 0 ? min(s.n_tiles, last / kBN + 1 - skip) : 0;
    ga = max(s.ns_tiles, (window_begin(first + n_tok - 1, cp.a.window) + kBN - 1) / kBN - skip);
    gb = min(s.n_tiles, min(first + 1, s.end) / kBN - skip);
    gs = min(s.ns_tiles, min(cp.a.n_sink, min(first + 1, s.end)) / kBN);
    if (n_tok == 0 || last < 0) ex = 0, gs = gb = 0;
  }
  __device__ __forceinline__ bool sees(int i, int ns_tiles) const { return ex > 0 && (i < ns_tiles || (i >= fx && i < ex)); }
  __device__ __forceinline__ bool sees_all(int i) const { return i < gs || (i >= ga && i < gb); }
};

// A warp's place in its CTA's share.  It lives in shared memory, one per warp: the registers belong to the
// products and weights.  One lane moves it.
struct Walk {
  int b, blk, n_blk, kvh, i0, i1, left;
  Block s;
  Half hx[2];
  __device__ __forceinline__ void block(const Q8ChunkParams &cp) {
    s = block_of(cp, b, blk);
    hx[0].of(cp, s, 0);
    hx[1].of(cp, s, 1);
  }
  // `offset`: the share's begin on the runs of this block's KV heads; a run is kPieceCost, then its tiles
  __device__ __forceinline__ bool begin(const Q8ChunkParams &cp, int b_, int blk_, int offset, int share) {
    b = b_, blk = blk_;
    n_blk = blocks_of(cp, b);
    block(cp);
    kvh = offset / (s.n_tiles + kPieceCost);
    const int at = offset - kvh * (s.n_tiles + kPieceCost);
    i0 = max(0, at - kPieceCost);
    left = share - max(0, kPieceCost - at);
    i1 = min(s.n_tiles, i0 + left);
    return left > 0;
  }
  __device__ __forceinline__ bool next(const Q8ChunkParams &cp) {
    left -= i1 - i0;
    if (left <= 0) return false;
    if (++kvh == cp.a.c.n_kv_heads) {
      kvh = 0;
      do {
        if (++blk >= n_blk) {
          blk = 0;
          do {
            if (++b >= cp.a.c.batch) return false;
            n_blk = blocks_of(cp, b);
          } while (n_blk == 0);
        }
        block(cp);
      } while (s.n_tiles == 0);
    }
    left -= kPieceCost;
    i0 = 0;
    i1 = min(s.n_tiles, left);
    return left > 0;
  }
};
__device__ __forceinline__ bool next_piece(Walk &w, const Q8ChunkParams &cp, int lane) { // all lanes
  __syncwarp();
  int more = 0;
  if (lane == 0) more = w.next(cp);
  __syncwarp();
  return __shfl_sync(0xffffffffu, more, 0) != 0;
}

// mbar_wait with the waiting itself out of the way of the instructions that follow
__device__ __forceinline__ bool await(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag, int *error_flag, int code) {
  if (__builtin_expect(mbar_try_wait(bar, parity), 1)) return true;
  return mbar_wait(bar, parity, abort_flag, error_flag, code);
}

__device__ __forceinline__ int block_scan(int mine, int *scratch, int warp, int lane, int &total) { // exclusive; all threads
  int incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  int before = incl - mine;
  total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    const int v = scratch[w];
    if (w < warp) before += v;
    total += v;
  }
  __syncthreads();
  return before;
}

static_assert(sizeof(Walk) <= kWalkBytes, "a warp's walk");

} // namespace q8c

template <typename T>
__global__ void __launch_bounds__(q8c::kThreads, 1)
attn_q8_chunk_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Q8ChunkParams cp) {
  using namespace q8c;
  const Q8AttnParams &p = cp.a;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t smem_base = smem_u32(smem);
  int *scan = reinterpret_cast<int *>(smem + kSmemScan);
  volatile int *refs = reinterpret_cast<volatile int *>(smem + kSmemRef);
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem + kSmemBar + BAR_COUNT * 8);
  volatile uint32_t *abort_flag = tmem_slot + 1;
  auto bar = [&](int i) { return smem_base + kSmemBar + 8u * i; };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = p.group, kvH = p.c.n_kv_heads, tok2 = 2 * cp.tile_tokens;
  int *err = p.c.error_flag;

  cudaTriggerProgrammaticLaunchCompletion();
  if (tid == 0) {
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(BAR_RAWFULL + s), 1);
      mbar_init(bar(BAR_RAWEMPTY + s), 4);
      mbar_init(bar(BAR_KFULL + s), 4);
      mbar_init(bar(BAR_KEMPTY + s), 2);
      mbar_init(bar(BAR_VFULL + s), 4);
      mbar_init(bar(BAR_VEMPTY + s), 2);
      mbar_init(bar(BAR_QFULL + s), 128);
      mbar_init(bar(BAR_QTAKEN + s), 1);
      mbar_init(bar(BAR_SFULL + s), 1);
      mbar_init(bar(BAR_SFREE + s), 128);
      for (int h = 0; h < 2; ++h) {
        mbar_init(bar(BAR_PFULL + 2 * h + s), 128);
        mbar_init(bar(BAR_ODONE + 2 * h + s), 1);
      }
    }
    for (int s = 0; s < 4; ++s) mbar_init(bar(BAR_REF + s), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  cudaGridDependencySynchronize();

  // ---- this CTA's share.  Blocks before each sequence (in the Q tiles), then tiles before each block.
  int *prefix = reinterpret_cast<int *>(smem + kSmemQ);
  int n_blocks;
  {
    const int per = (p.c.batch + kThreads - 1) / kThreads;
    const int lo = min(p.c.batch, tid * per), hi = min(p.c.batch, lo + per);
    int mine = 0;
    int falls = 0; // tok_start decreases somewhere: the rows overlap, and nothing below is sized for that
    for (int b = lo; b < hi; ++b) {
      mine += blocks_of(cp, b);
      falls |= __ldg(p.r.tok_start + b + 1) < __ldg(p.r.tok_start + b);
    }
    falls = __syncthreads_or(falls);
    if (falls) {
      if (tid == 0) report(err, kStatusOutsideCache);
      if (tid == 0 && blockIdx.x == 0) cp.head->n_blocks = 0;
      return;
    }
    int at = block_scan(mine, scan, warp, lane, n_blocks);
    for (int b = lo; b < hi; ++b) {
      prefix[b] = at;
      at += blocks_of(cp, b);
    }
    if (tid == 0) prefix[p.c.batch] = n_blocks;
    __syncthreads();
  }
  const int per = (n_blocks + kThreads - 1) / kThreads;
  const int u_lo = min(n_blocks, tid * per), u_hi = min(n_blocks, u_lo + per);
  int b_lo = 0;
  if (u_lo < u_hi) { // the sequence of block u_lo: the last one with prefix <= u_lo
    int len = p.c.batch;
    while (len > 1) {
      const int half = len / 2;
      if (prefix[b_lo + half] <= u_lo) b_lo += half;
      len -= half;
    }
  }
  int mine = 0;
  for (int u = u_lo, b = b_lo; u < u_hi; ++u) {
    while (u >= prefix[b + 1]) ++b;
    const int tiles = block_of(cp, b, u - prefix[b]).n_tiles;
    mine += tiles > 0 ? tiles + kPieceCost : 0;
  }
  int total;
  const int before = block_scan(mine, scan, warp, lane, total);
  const long W = static_cast<long>(total) * kvH;
  const int n = static_cast<int>(min(static_cast<long>(gridDim.x), W));
  const int c = blockIdx.x;
  const long x0 = c < n ? share_begin(W, n, c) : -1, x1 = c < n ? share_begin(W, n, c + 1) : -1;
  if (c == 0 && tid == 0) cp.head->n_blocks = n_blocks;
  {
    long at = static_cast<long>(before) * kvH;
    for (int u = u_lo, b = b_lo; u < u_hi; ++u) {
      while (u >= prefix[b + 1]) ++b;
      const Block s = block_of(cp, b, u - prefix[b]);
      const int one = s.n_tiles > 0 ? s.n_tiles + kPieceCost : 0;
      const long run = static_cast<long>(one) * kvH;
      if (x0 >= at && x0 < at + run) {
        scan[16] = b;
        scan[17] = u - prefix[b];
        scan[18] = static_cast<int>(x0 - at);
      }
      // the CTAs share the writing of the merge's records: this one has those of number c, c + grid, ...
      const int ctas = static_cast<int>(gridDim.x), ahead = c - static_cast<int>(static_cast<unsigned>(u) * kvH % gridDim.x);
      for (int h = ahead < 0 ? ahead + ctas : ahead; h < kvH; h += ctas) {
        RunInfo r{};
        r.c1 = -1;
        if (s.n_tiles > 0) {
          const long first = at + static_cast<long>(h) * one;
          r.c0 = share_of(W, n, first + kPieceCost);
          r.c1 = share_of(W, n, first + one - 1);
            r.slot0 = 2 * r.c0 + (share_begin(W, n, r.c0) >= first ? 0 : 1);
        }
        r.t0 = s.t0;
        r.nq = s.nq;
        cp.info[static_cast<long>(u) * kvH + h] = r;
      }
      at += run;
    }
  }
  if ((smem_base & 1023u) != 0 && tid == 0) report(err, 30);
  __syncthreads();
  if (c >= n || (smem_base & 1023u) != 0) return;
  const int b_first = scan[16], blk_first = scan[17], off_first = scan[18], share = static_cast<int>(x1 - x0);
  Walk &w = *reinterpret_cast<Walk *>(smem + kSmemWalk + warp * kWalkBytes);
  int some = 0;
  if (lane == 0) some = w.begin(cp, b_first, blk_first, off_first, share);
  if (!__syncthreads_or(some)) return; // the share is all cost and no tile
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t *>(tmem_slot))), "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads(); // also: the prefix sums in the Q tiles are done with
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 4) {
    reg_dec<96>();
    if (warp == 0) {
      // ---------------------------------------------------------- TMA producer
      uint32_t g = 0;
      bool ok = true;
      do {
        for (int base = w.i0; base < w.i1 && ok; base += 16) {
          // lanes 2 k, 2 k + 1: the two halves of the k-th tile from here: page, row in it, and whether anyone sees it
          int outer = w.b, row = 0;
          bool on = false;
          if (base + (lane >> 1) < w.i1) {
            row = w.s.tile(base + (lane >> 1)) * kBN + 64 * (lane & 1);
            on = row < w.s.end && (row + 64 > w.s.lo || row < w.s.ns);
            if (on && p.c.pg.table) {
              outer = __ldg(p.c.pg.table + static_cast<long>(w.b) * p.c.pg.table_stride + (row >> p.c.pg.page_shift));
              row &= (1 << p.c.pg.page_shift) - 1;
              if (static_cast<unsigned>(outer) >= static_cast<unsigned>(p.c.pg.n_pages)) {
                report(err, kStatusOutsideCache);
                outer = 0;
              }
            }
          }
          const int cnt = min(16, w.i1 - base);
          for (int k = 0; k < cnt && ok; ++k, ++g) {
            int o[2], r[2];
            bool live[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              o[h] = __shfl_sync(0xffffffffu, outer, 2 * k + h);
              r[h] = __shfl_sync(0xffffffffu, row, 2 * k + h);
              live[h] = __shfl_sync(0xffffffffu, static_cast<int>(on), 2 * k + h) != 0;
            }
            if (lane == 0) {
#pragma unroll
              for (int kv = 0; kv < 2; ++kv) {
                ok = ok && await(bar(BAR_RAWEMPTY + kv), (g & 1) ^ 1, abort_flag, err, 1);
                if (!ok) break;
                const uint32_t full = bar(BAR_RAWFULL + kv);
                uint32_t bytes = 0, xb[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  // exponent rows of a flat cache end at max_pos rounded up to 16
                  xb[h] = p.c.pg.table ? 64u : static_cast<uint32_t>(min(64, ((p.c.max_pos + 15) & ~15) - r[h]));
                  if (live[h]) bytes += 64 * 128 + (kv == 0 ? 2 * xb[h] : 0);
                }
                mbar_expect_tx(full, bytes);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  if (!live[h]) continue;
                  tma_load_4d(smem_base + kSmemRaw + kv * kRawBytes + h * 64 * 128, kv ? &map_v : &map_k, full, 0, r[h], w.kvh, o[h]);
                  if (kv == 0) { // the exponents of V come along: the softmax needs their largest with K
                    const long xo = static_cast<long>(o[h]) * p.c.x_outer + w.kvh * p.c.x_head + r[h];
                    bulk_load(smem_base + kSmemExp + 64 * h, p.c.kx + xo, xb[h], full);
                    bulk_load(smem_base + kSmemExp + 128 + 64 * h, p.c.vx + xo, xb[h], full);
                  }
                }
              }
            }
            ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0) != 0;
          }
        }
      } while (ok && next_piece(w, cp, lane));
    } else if (warp < 3) {
      // ---------------------------------------------------------- MMA issuer of tile X
      // One warp each for A and B.  A tile is taken in two steps of 64 positions.  The softmax warps
      // copy a step's scores to registers and free them at once, so that the next step's scores are
      // made while they work: Q.K of step n + 1 goes before P.V of step n.
      // The whole warp walks through this, on values that are visibly the same in all lanes, and one
      // elected lane issues: the descriptors then live in uniform registers, from where the products
      // take them; a lone lane has to move six values there for each product.
      const int x = __shfl_sync(0xffffffffu, warp, 0) - 1;
      constexpr uint32_t idesc_qk = (instr_desc(0u, 0) & ~(0x3fu << 17)) | ((64u >> 3) << 17), idesc_pv = instr_desc(0u, 1);
      constexpr uint32_t kTileStep = kTileBytes >> 4, kHalfStep = kHalfTile >> 4, kRows64 = (64 * 128) >> 4;
      const uint32_t base_u = __shfl_sync(0xffffffffu, smem_base, 0), tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t dq0 = smem_desc_lo(base_u + kSmemQ, 16) + x * kTileStep;
      const uint32_t dk0 = smem_desc_lo(base_u + kSmemK, 16);
      const uint32_t dv0 = smem_desc_lo(base_u + kSmemV, kHalfTile);
      const uint32_t scol = tmem_u + kColS + 64 * x, pcol = tmem_u + kColP + 64 * x, ocol = tmem_u + kColO + 128 * x;
      const uint32_t bars = base_u + kSmemBar;
      auto ubar = [&](int i) { return bars + 8u * i; };
      auto wait = [&](int i, uint32_t parity, int code) -> bool {
        return __all_sync(0xffffffffu, await(ubar(i), parity, abort_flag, err, code));
      };
      const bool leader = elect_one();
      uint32_t gk = 0, gv = 0;        // tiles of the share whose K, whose V has been used
      uint32_t nqk = 0, npv = 0;      // steps so far
      uint32_t piece = 0;
      bool ok = true;
      do {
        const int i0 = __shfl_sync(0xffffffffu, w.i0, 0), i1 = __shfl_sync(0xffffffffu, w.i1, 0), ns_tiles = __shfl_sync(0xffffffffu, w.s.ns_tiles, 0);
        const int fx = __shfl_sync(0xffffffffu, w.hx[x].fx, 0), ex = __shfl_sync(0xffffffffu, w.hx[x].ex, 0);
        // the rows of Q; their writers have also taken the previous piece's results out
        ok = wait(BAR_QFULL + x, piece & 1, 3);
        if (!ok) break;
        if (leader) mbar_arrive(ubar(BAR_QTAKEN + x));
        uint32_t acc = 0, h = 0, ph = 0;
        bool pending = false;          // a step whose scores have been issued, but not its P.V
        for (int i = i0; i <= i1;) {
          const bool more = i < i1, on = more && ex > 0 && (i < ns_tiles || (i >= fx && i < ex));
          if (on) {                    // S = Q.K of step h
            const uint32_t s = gk & 1;
            if (h == 0) ok = wait(BAR_KFULL + s, (gk >> 1) & 1, 4);
            ok = ok && wait(BAR_SFREE + x, (nqk & 1) ^ 1, 11);
            if (!ok) break;
            tc_fence_after();
            const uint32_t dk = dk0 + s * kTileStep + h * kRows64;
            if (leader) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const uint32_t ko = (k >> 2) * kHalfStep + (k & 3) * 2;
                tc_mma_ss(scol, dq0 + ko, dk + ko, kDescHi, idesc_qk, k > 0);
              }
              tc_commit(ubar(BAR_SFULL + x));
              if (h) tc_commit(ubar(BAR_KEMPTY + s)); // arrives when the products issued so far have read their operands
            }
            __syncwarp();
            ++nqk;
          }
          if (pending) {               // O += P.V of the step before
            const uint32_t s = gv & 1;
            if (ph == 0) ok = wait(BAR_VFULL + s, (gv >> 1) & 1, 6);
            ok = ok && wait(BAR_PFULL + 2 * ph + x, (npv >> 1) & 1, 10);
            if (!ok) break;
            tc_fence_after();
            const uint32_t dv = dv0 + s * kTileStep + ph * kRows64, pc = pcol + 32 * ph;
            if (leader) {
#pragma unroll
              for (int k = 0; k < 4; ++k) tc_mma_ts(ocol, pc + 8 * k, dv + k * (2048 >> 4), kDescHi, idesc_pv, k > 0 ? 1u : acc);
              tc_commit(ubar(BAR_ODONE + 2 * ph + x));
              if (ph) tc_commit(ubar(BAR_VEMPTY + s));
            }
            __syncwarp();
            acc = 1u;
            ++npv;
            gv += ph;
          }
          pending = on;
          ph = h;
          if (on) {
            gk += h;
            i += static_cast<int>(h);
            h ^= 1u;
          } else {
            if (more) {                // a tile that X has no use for
              ok = wait(BAR_KFULL + (gk & 1), (gk >> 1) & 1, 5) && wait(BAR_VFULL + (gv & 1), (gv >> 1) & 1, 5);
              if (!ok) break;
              if (leader) {
                mbar_arrive(ubar(BAR_KEMPTY + (gk & 1)));
                mbar_arrive(ubar(BAR_VEMPTY + (gv & 1)));
              }
              ++gk;
              ++gv;
            }
            ++i;
          }
        }
        ++piece;
      } while (ok && next_piece(w, cp, lane));
    }
  } else if (warp < 12) {
    reg_inc<152>();
    // ------------------------------------------------------------ softmax, Q and results of tile X
    const int x = (warp >> 2) - 1, quad = warp & 3;
    const int r = quad * 32 + lane;              // row of the tile
    const int tok = r / G, hd = r - tok * G;     // its token and head of the group
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t scol = tmem + lane_addr + kColS + 64 * x, pcol = tmem + lane_addr + kColP + 64 * x, ocol = tmem + lane_addr + kColO + 128 * x;
    uint32_t g = 0, cnt = 0;
    int piece = 0;
    bool ok = true;
    do {
      const Half &hx = w.hx[x];
      const bool live = tok < hx.n_tok;          // tok < tile_tokens for every row that exists
      const long t = static_cast<long>(w.s.t0) + x * cp.tile_tokens + tok;
      // a tile that sees nothing of a piece must not run more than one piece ahead of the MMA warp
      if (piece > 0 && !__all_sync(0xffffffffu, await(bar(BAR_QTAKEN + x), (piece - 1) & 1, abort_flag, err, 13))) break;
      // ---- the row of Q, scaled to fp16: its largest magnitude to 2^13 .. 2^14
      float rowc, up;
      {
        const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const T *>(p.q) + t * p.q_row + (w.kvh * G + hd) * kHeadDim);
        uint32_t top = 0;
#pragma unroll 1
        for (int i = 0; i < 16; i += 8) {
          uint4 u[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) u[k] = live ? src[i + k] : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            // magnitudes of 16-bit floats order like their bit patterns
            top = __vmaxu2(top, __vmaxu2(__vmaxu2(u[k].x & 0x7fff7fffu, u[k].y & 0x7fff7fffu), __vmaxu2(u[k].z & 0x7fff7fffu, u[k].w & 0x7fff7fffu)));
          }
        }
        const float2 two = Elem<T>::unpack(max(top & 0xffffu, top >> 16));
        const uint32_t topf = __float_as_uint(two.x) & 0x7fffffffu;
        int e = max(static_cast<int>(topf >> 23) - 127, -100);
        if (topf >= 0x7f800000u) e = 13;         // not finite: as it is
        up = pow2i(13 - e);
        rowc = p.scale_log2 * pow2i(e - 13);
        const uint32_t dst = smem_base + kSmemQ + x * kTileBytes + r * 128;
#pragma unroll 1
        for (int i = 0; i < 16; i += 4) {
          uint4 u[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) u[k] = live ? src[i + k] : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t *wd = reinterpret_cast<uint32_t *>(&u[k]);
#pragma unroll
            for (int e2 = 0; e2 < 4; ++e2) {
              const float2 v = Elem<T>::unpack(wd[e2]);
              wd[e2] = Elem<__half>::pack(v.x * up, v.y * up);
            }
            const uint32_t chunk = static_cast<uint32_t>((i + k) & 7) ^ static_cast<uint32_t>(r & 7);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (i >> 3) * kHalfTile + (chunk << 4)), "r"(u[k].x), "r"(u[k].y),
                         "r"(u[k].z), "r"(u[k].w)
                         : "memory");
          }
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(bar(BAR_QFULL + x));

      const int pos = hx.first + tok;
      const int vend = live ? min(pos + 1, w.s.end) : 0, wlo = window_begin(pos, p.window);
      const int i0 = w.i0, i1 = w.i1, ns_tiles = w.s.ns_tiles, skip = w.s.w0 - ns_tiles;
      const int fx = hx.fx, ex = hx.ex, ga = hx.ga, gb = hx.gb, gs = hx.gs;
      float m_ref = -INFINITY, l = 0.f;
      bool begun = false;
      for (int i = i0; i < i1; ++i, ++g) {
        if (!(ex > 0 && (i < ns_tiles || (i >= fx && i < ex)))) continue;
        const bool all = i < gs || (i >= ga && i < gb);     // every row sees all of the tile
        const int col0 = (i < ns_tiles ? i : i + skip) * kBN;
        float a = 0.f, off = 0.f, inv_v = 0.f;
#pragma unroll 1
        for (uint32_t h = 0; h < 2; ++h, ++cnt) {
          ok = ok && await(bar(BAR_SFULL + x), cnt & 1, abort_flag, err, 7);
          if (h == 0) ok = ok && await(bar(BAR_REF + (g & 3)), (g >> 2) & 1, abort_flag, err, 12); // complete by now: K was converted before S
          // this half of P was last read by the product two steps ago: almost always done by now, asked early
          uint32_t p_free = cnt < 2 || mbar_try_wait(bar(BAR_ODONE + 2 * h + x), ((cnt - 2) >> 1) & 1);
          if (__builtin_expect(!__all_sync(0xffffffffu, ok), 0)) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t su[64];
          tc_ld32(scol, su);
          tc_ld32(scol + 32, su + 32);
          if (h == 0) {
            const int rk = refs[2 * (g & 3)], rv = refs[2 * (g & 3) + 1];
            a = fmaxf(rowc * pow2i(rk - 7), 1.2e-38f);
            off = static_cast<float>(rv - 7);
            inv_v = pow2i(7 - rv);
          }
          tc_wait_ld();
          tc_fence_before();
          mbar_arrive(bar(BAR_SFREE + x));   // the scores are in registers: the next step's may come
          if (__builtin_expect(!all, 0)) { // hide what the row does not see
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int c0 = col0 + 64 * static_cast<int>(h) + 32 * q;
              auto below = [&](int k) { return k - c0 <= 0 ? 0u : k - c0 >= 32 ? 0xffffffffu : (1u << (k - c0)) - 1u; }; // columns < k
              const uint32_t vis = below(vend) & (~below(wlo) | below(p.n_sink));
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!(vis & (1u << j))) su[32 * q + j] = 0xff800000u; // -inf
            }
          }
          float mxa[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) mxa[k] = fmaxf(__uint_as_float(su[k]), __uint_as_float(su[8 + k]));
#pragma unroll
          for (int j = 16; j < 64; j += 16) {
#pragma unroll
            for (int k = 0; k < 8; ++k) mxa[k] = max3(mxa[k], __uint_as_float(su[j + k]), __uint_as_float(su[j + 8 + k]));
          }
          const float mx = fmaf(fmaxf(max3(mxa[0], mxa[1], mxa[2]), max3(max3(mxa[3], mxa[4], mxa[5]), mxa[6], mxa[7])), a, off);
          const bool grow = mx > m_ref + kLazy;
          if (__builtin_expect(__any_sync(0xffffffffu, grow) && begun, 0)) {
            // O must hold every product issued so far: those of this half's last step and of the other's
            ok = await(bar(BAR_ODONE + 2 * (h ^ 1) + x), ((cnt - 1) >> 1) & 1, abort_flag, err, 8);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const float f = grow ? ex2(m_ref - mx) : 1.f;
            l *= f;
#pragma unroll 1
            for (int q4 = 0; q4 < 4; ++q4) {
              uint32_t o[32];
              tc_ld32(ocol + 32 * q4, o);
              tc_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tc_st32(ocol + 32 * q4, o);
            }
            tc_wait_st();
          }
          if (grow) m_ref = mx;
          begun = true;
          const float nm = off - (m_ref == -INFINITY ? 0.f : m_ref); // nothing seen yet: P = 0
          uint64_t sums[2] = {0ull, 0ull};
          const uint64_t a2 = pack2(a, a), nm2 = pack2(nm, nm);
          uint32_t pk[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const uint64_t y2 = fma2(pack2(__uint_as_float(su[2 * j]), __uint_as_float(su[2 * j + 1])), a2, nm2);
            float y0, y1;
            unpack2(y2, y0, y1);
            const float e0 = ex2(y0), e1 = ex2(y1);
            sums[j & 1] = add2(sums[j & 1], pack2(e0, e1));
            pk[j] = Elem<__half>::pack(e0, e1);
          }
          if (__builtin_expect(!__all_sync(0xffffffffu, p_free), 0)) {
            ok = await(bar(BAR_ODONE + 2 * h + x), ((cnt - 2) >> 1) & 1, abort_flag, err, 14);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
          }
          tc_st32(pcol + 32 * h, pk);
          float s0, s1, s2, s3;
          unpack2(sums[0], s0, s1);
          unpack2(sums[1], s2, s3);
          l = fmaf((s0 + s1) + (s2 + s3), inv_v, l);
          tc_wait_st();
          tc_fence_before();
          mbar_arrive(bar(BAR_PFULL + 2 * h + x));
        }
        if (!ok) break;
      }
      if (!ok) break;
      // ---- the piece's result
      if (begun && !__all_sync(0xffffffffu, await(bar(BAR_ODONE + 2 + x), ((cnt - 1) >> 1) & 1, abort_flag, err, 9))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const bool whole = w.i0 == 0 && w.i1 == w.s.n_tiles;
      const float inv = l == 0.f ? 0.f : 1.f / l;  // NaN stays NaN
      const long slot_row = static_cast<long>(2 * c + (piece == 0 ? 0 : 1)) * (tok2 * G) + (x * cp.tile_tokens + tok) * G + hd;
      T *dst = static_cast<T *>(p.out) + t * p.out_row + (w.kvh * G + hd) * kHeadDim;
#pragma unroll 1
      for (int q4 = 0; q4 < 4; ++q4) {
        uint32_t o[32];
        if (begun) {
          tc_ld32(ocol + 32 * q4, o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0u;
        }
        if (live && whole) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 v;
            v.x = Elem<T>::pack(__uint_as_float(o[8 * j]) * inv, __uint_as_float(o[8 * j + 1]) * inv);
            v.y = Elem<T>::pack(__uint_as_float(o[8 * j + 2]) * inv, __uint_as_float(o[8 * j + 3]) * inv);
            v.z = Elem<T>::pack(__uint_as_float(o[8 * j + 4]) * inv, __uint_as_float(o[8 * j + 5]) * inv);
            v.w = Elem<T>::pack(__uint_as_float(o[8 * j + 6]) * inv, __uint_as_float(o[8 * j + 7]) * inv);
            reinterpret_cast<uint4 *>(dst)[4 * q4 + j] = v;
          }
        } else if (live) {
          float4 *part = reinterpret_cast<float4 *>(cp.o + slot_row * kHeadDim);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            part[8 * q4 + j] = make_float4(__uint_as_float(o[4 * j]) * inv, __uint_as_float(o[4 * j + 1]) * inv,
                                           __uint_as_float(o[4 * j + 2]) * inv, __uint_as_float(o[4 * j + 3]) * inv);
        }
        __syncwarp(); // tcgen05.ld takes the whole warp
      }
      if (live && !whole) cp.lse[slot_row] = l == 0.f ? -INFINITY : (m_ref == -INFINITY ? 0.f : m_ref) + log2f(l);
      ++piece;
    } while (next_piece(w, cp, lane));
  } else {
    reg_dec<112>();
    // ------------------------------------------------------------ converters: 32 rows of every tile per warp
    const int cw = warp - 12;
    uint32_t g = 0;
    bool ok = true;
    // Rows 32 cw .. 32 cw + 31 of the raw tile -> fp16 operand tile.  `f`: this lane's row's factor, two
    // fp16 (0: a row that nobody sees, written as zeros).  Eight lanes access shared memory at once: four
    // 16-byte pieces of the codes of row a and of row a ^ 5, which the 128-byte swizzle of the codes puts
    // into eight different bank groups, and that of the operand tile as well.
    const int pr = (lane >> 3) ^ ((lane & 4) ? 5 : 0);
    auto convert = [&](uint32_t raw, uint32_t dst, uint32_t f) {
      const bool hole = __any_sync(0xffffffffu, f == 0u);
      uint32_t wv[8][4], fr[4];
#pragma unroll
      for (int b8 = 0; b8 < 4; ++b8) {       // eight rows, both 64-element halves
        const int rl = b8 * 8 + pr, row = 32 * cw + rl, sw = row & 7;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(wv[2 * b8 + h][0]), "=r"(wv[2 * b8 + h][1]), "=r"(wv[2 * b8 + h][2]), "=r"(wv[2 * b8 + h][3])
                       : "r"(raw + row * 128 + (((4 * h + (lane & 3)) ^ sw) << 4)));
        fr[b8] = __shfl_sync(0xffffffffu, f, rl);
      }
      if (__builtin_expect(hole, 0)) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (fr[e >> 3] == 0u) wv[e >> 2][e & 3] = 0u; // whatever the bytes are
      }
#pragma unroll
      for (int b8 = 0; b8 < 4; ++b8) {
        const int row = 32 * cw + b8 * 8 + pr, sw = row & 7;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t o[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            cvt_e4m3x4_f16x4(wv[2 * b8 + h][e], o[2 * e], o[2 * e + 1]);
            o[2 * e] = hmul2(o[2 * e], fr[b8]);
            o[2 * e + 1] = hmul2(o[2 * e + 1], fr[b8]);
          }
          const uint32_t base = dst + h * kHalfTile + row * 128, c0 = 2 * (lane & 3);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + ((c0 ^ sw) << 4)), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + (((c0 + 1) ^ sw) << 4)), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
        }
      }
    };
    // 2^(7 - d) as two fp16; d: how far the row's exponent lies below the tile's largest
    auto factor = [](int d) -> uint32_t {
      const uint32_t h = d <= 21 ? static_cast<uint32_t>(15 + 7 - d) << 10 : d <= 31 ? 1u << (31 - d) : 0u;
      return h | (h << 16);
    };
    do {
      for (int i = w.i0; ok && i < w.i1; ++i, ++g) {
        const int col0 = w.s.tile(i) * kBN;
        const uint32_t ph = g & 1, s = g & 1, sph = (g >> 1) & 1;
        ok = await(bar(BAR_RAWFULL + 0), ph, abort_flag, err, 20);
        if (!__all_sync(0xffffffffu, ok)) break;
        // the largest exponents among the rows that someone sees (every warp for itself: 4 rows a lane)
        const uint32_t kx4 = *reinterpret_cast<const uint32_t *>(smem + kSmemExp + 4 * lane);
        const uint32_t vx4 = *reinterpret_cast<const uint32_t *>(smem + kSmemExp + 128 + 4 * lane);
        auto seen = [&](int j) { return j < w.s.end && (j >= w.s.lo || j < w.s.ns); };
        int rk = 0, rv = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kx = (kx4 >> (8 * e)) & 0xff, vx = (vx4 >> (8 * e)) & 0xff;
          if (seen(col0 + 4 * lane + e) && kx != kPoison && vx != kPoison) rk = max(rk, kx), rv = max(rv, vx);
        }
        rk = __reduce_max_sync(0xffffffffu, rk);
        rv = __reduce_max_sync(0xffffffffu, rv);
        const int row = 32 * cw + lane;
        const int kx = smem[kSmemExp + row], vx = smem[kSmemExp + 128 + row];
        const bool vis = seen(col0 + row), poison = kx == kPoison || vx == kPoison;
        const uint32_t fk = !vis ? 0u : poison ? 0x7e007e00u : factor(rk - kx);
        const uint32_t fv = !vis || poison ? 0u : factor(rv - vx);
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          if (kv) ok = await(bar(BAR_RAWFULL + 1), ph, abort_flag, err, 22);
          ok = ok && await(bar((kv ? BAR_VEMPTY : BAR_KEMPTY) + s), sph ^ 1, abort_flag, err, 21);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          convert(smem_base + kSmemRaw + kv * kRawBytes, smem_base + (kv ? kSmemV : kSmemK) + s * kTileBytes, kv ? fv : fk);
          if (kv == 0 && cw == 0 && lane == 0) {
            refs[2 * (g & 3)] = rk - 127;
            refs[2 * (g & 3) + 1] = rv - 127;
            mbar_arrive(bar(BAR_REF + (g & 3)));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(bar((kv ? BAR_VFULL : BAR_KFULL) + s));
            mbar_arrive(bar(BAR_RAWEMPTY + kv));
          }
        }
      }
    } while (__all_sync(0xffffffffu, ok) && next_piece(w, cp, lane));
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// Merges the pieces of the blocks that were cut, and zeroes the rows that see nothing.
template <typename T> __global__ void __launch_bounds__(32 * kMergeWarps) attn_q8_chunk_merge_kernel(const Q8ChunkParams cp, int split) {
  using namespace q8c;
  const Q8AttnParams &p = cp.a;
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
  const int kvH = p.c.n_kv_heads, G = p.group;
  const int u = blockIdx.x / kvH, kvh = blockIdx.x - u * kvH;
  if (u >= cp.head->n_blocks) return;
  const RunInfo info = cp.info[blockIdx.x];
  if (info.c1 == info.c0) return; // one CTA did the whole block
  const int block_rows = 2 * cp.tile_tokens * G;
  merge_rows(cp.o, cp.lse, info.c1 - info.c0 + 1, info.nq * G, split,
             [&](int i, int rho) { return static_cast<long>(i == 0 ? info.slot0 : 2 * (info.c0 + i)) * block_rows + rho; },
             [&](int rho, const float4 &v) {
               const int tok = rho / G;
               uint2 o;
               o.x = Elem<T>::pack(v.x, v.y);
               o.y = Elem<T>::pack(v.z, v.w);
               *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + (static_cast<long>(info.t0) + tok) * p.out_row +
                                          (kvh * G + rho - tok * G) * kHeadDim + (threadIdx.x & 31) * 4) = o;
             });
}

namespace {

// Blocks a batch can have at most, and CTAs to launch.
long block_bound(int batch, int group, int total) {
  const int tok2 = 2 * (128 / group);
  return total / tok2 + (batch < total ? batch : total);
}
int chunk_ctas(int batch, int n_kv_heads, int group, int total, int max_kv_len) {
  const long tiles = block_bound(batch, group, total) * n_kv_heads * ((static_cast<long>(max_kv_len) + q8c::kBN - 1) / q8c::kBN);
  return static_cast<int>(tiles < q8c::kMaxCtas ? tiles : q8c::kMaxCtas);
}

template <typename T> cudaError_t launch_typed(const Q8ChunkParams &cp, const CUtensorMap &mk, const CUtensorMap &mv, int n_ctas, long blocks, cudaStream_t stream, int *launches) {
  // the shared-memory opt-in is a property of (function, device): set on the first launch per device
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !done[dev]) {
    e = cudaFuncSetAttribute(attn_q8_chunk_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, q8c::kSmemTotal);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  e = launch_dependent(attn_q8_chunk_kernel<T>, dim3(n_ctas), q8c::kThreads, q8c::kSmemTotal, stream, mk, mv, cp);
  if (e != cudaSuccess) return e;
  *launches = 1;
  dim3 grid;
  int split;
  merge_shape(blocks * cp.a.c.n_kv_heads, 2 * cp.tile_tokens * cp.a.group, n_ctas, &grid, &split);
  e = launch_dependent(attn_q8_chunk_merge_kernel<T>, grid, 32 * kMergeWarps, 0, stream, cp, split);
  if (e != cudaSuccess) return e;
  *launches = 2;
  return cudaGetLastError();
}

} // namespace

size_t attn_q8_chunk_ws_bytes(int batch, int n_kv_heads, int group, int total, int max_kv_len) {
  const size_t rows = 2 * static_cast<size_t>(chunk_ctas(batch, n_kv_heads, group, total, max_kv_len)) * (2 * (128 / group) * group);
  return sizeof(q8c::Head) + static_cast<size_t>(block_bound(batch, group, total)) * n_kv_heads * sizeof(q8c::RunInfo) +
         rows * (kHeadDim + 1) * sizeof(float);
}

cudaError_t launch_attn_q8_chunk(const Q8AttnParams &p, bool bf16, cudaStream_t stream, int *launches) {
  *launches = 0;
  const Q8Cache &c = p.c;
  Q8ChunkParams cp{};
  cp.a = p;
  cp.tile_tokens = 128 / p.group;
  const int n_ctas = chunk_ctas(c.batch, c.n_kv_heads, p.group, p.r.total, p.max_kv_len);
  const long blocks = block_bound(c.batch, p.group, p.r.total);
  char *ws = static_cast<char *>(p.ws);
  cp.head = reinterpret_cast<q8c::Head *>(ws);
  cp.info = reinterpret_cast<q8c::RunInfo *>(ws + sizeof(q8c::Head));
  cp.o = reinterpret_cast<float *>(ws + sizeof(q8c::Head) + static_cast<size_t>(blocks) * c.n_kv_heads * sizeof(q8c::RunInfo));
  cp.lse = cp.o + 2 * static_cast<size_t>(n_ctas) * (2 * cp.tile_tokens * p.group) * kHeadDim;
  const uint64_t rows = c.pg.table ? 1ull << c.pg.page_shift : static_cast<uint64_t>(c.max_pos);
  const uint64_t outers = c.pg.table ? static_cast<uint64_t>(c.pg.n_pages) : static_cast<uint64_t>(c.batch);
  CUtensorMap mk, mv;
  if (!make_tensor_map_u8(&mk, true, c.k, rows, c.n_kv_heads, outers, c.c_pos, c.c_head, c.c_outer, 64) ||
      !make_tensor_map_u8(&mv, true, c.v, rows, c.n_kv_heads, outers, c.c_pos, c.c_head, c.c_outer, 64))
    return cudaErrorNotSupported;
  return bf16 ? launch_typed<__nv_bfloat16>(cp, mk, mv, n_ctas, blocks, stream, launches)
              : launch_typed<__half>(cp, mk, mv, n_ctas, blocks, stream, launches);
}

} // namespace b200attn
