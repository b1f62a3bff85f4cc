// Device helpers of the 8-bit KV cache: where a row lies, which sequence a token row belongs to, and
// the e4m3 <-> 16-bit conversions.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace b200attn {
namespace q8 {

constexpr int kMinExp = -100;    // smallest row exponent
constexpr int kPoison = 255;     // exponent byte of a row that holds a value that is not finite

__device__ __forceinline__ void report(int *error_flag, int code) {
  if (error_flag) *reinterpret_cast<volatile int *>(error_flag) = code;
}

// Outer index (sequence or page) and in-page position of position pos of sequence b; false if the
// position or its page lies outside the cache.
__device__ __forceinline__ bool locate(const Q8Cache &c, int b, int pos, long &outer, int &in_pos) {
  if (static_cast<unsigned>(pos) >= static_cast<unsigned>(c.max_pos)) return false;
  if (!c.pg.table) {
    outer = b;
    in_pos = pos;
    return true;
  }
  const int page = __ldg(c.pg.table + static_cast<long>(b) * c.pg.table_stride + (pos >> c.pg.page_shift));
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.pg.n_pages)) return false;
  outer = page;
  in_pos = pos & ((1 << c.pg.page_shift) - 1);
  return true;
}

// Sequence of token row t: the number of entries tok_start[1 .. batch] that are <= t, found by the
// eight threads of a group (`sub` 0 .. 7) together, eight probes a round.  All 32 lanes take part.
// batch: the row lies behind the last sequence.
__device__ __forceinline__ int seq_of_row(const int32_t *tok_start, int batch, int t, int lane) {
  const int sub = lane & 7, shift = lane & 24;
  int lo = 0, len = batch; // the count lies in [lo, lo + len]
  while (__any_sync(0xffffffffu, len > 0)) {
    const int step = (len + 7) >> 3;
    const int idx = lo + step * (sub + 1);
    const bool le = len > 0 && idx <= lo + len && __ldg(tok_start + idx) <= t;
    const int k = __popc((__ballot_sync(0xffffffffu, le) >> shift) & 0xffu);
    const int hi = min(lo + len, lo + step * (k + 1) - 1);
    lo += step * k;
    len = len > 0 ? max(0, hi - lo) : 0;
  }
  return lo;
}

__device__ __forceinline__ void lds128(uint32_t *r, uint32_t addr) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// An 8 x 8 block of 16-bit values held as a product's result (two neighbours of a row per lane), transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Four e4m3 codes -> two pairs of fp16 values, exact.  (Handed over as 16-bit halves the conversions take
// them from where they are; masked and shifted out first they cost half as much again: decode of long caches
// 327 us that way, 280 this way.)
__device__ __forceinline__ void cvt_e4m3x4_f16x4(uint32_t u, uint32_t &lo, uint32_t &hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(u));
}
// Two fp32 values -> two e4m3 codes (a in the low byte), to nearest even.
__device__ __forceinline__ uint32_t cvt_f32_e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); } // -126 <= e <= 127

// Exponent of a row whose largest magnitude is amax (finite): the smallest e >= kMinExp with
// amax <= 448 * 2^e = 1.75 * 2^(e + 8).  Adding what lies between 1.75 and 2 to the mantissa carries
// into the exponent field exactly when the mantissa is above 1.75.
__device__ __forceinline__ int row_exp(float amax) {
  const int e = static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
  return max(e, kMinExp);
}

// One query row's visible positions: [0, min(sink, lo)) and [lo, pos].
__device__ __forceinline__ int window_begin(int pos, int window) { return window > 0 ? max(0, pos - window + 1) : 0; }

// The tiles of TILE positions that a run of consecutive rows sees: those of the first positions, 0 ..
// ns_tiles - 1, and those from the first row's window to the last row, w0, w0 + 1, ...
template <int TILE> struct Span {
  int t0, nq;          // the first row and the number of rows
  int pos0;            // position of the first row
  int end;             // one past the last visible position
  int lo;              // first window position of the first row
  int ns;              // first positions visible besides the window
  int ns_tiles, w0, n_tiles;
  __device__ __forceinline__ int tile(int i) const { return i < ns_tiles ? i : w0 + i - ns_tiles; }
  __device__ __forceinline__ void cover(const Q8AttnParams &p, int limit) { // from t0, nq, pos0
    end = nq > 0 ? max(0, static_cast<int>(min(static_cast<long>(pos0) + nq, static_cast<long>(limit)))) : 0;
    lo = min(window_begin(pos0, p.window), end);
    ns = min(p.n_sink, lo);
    ns_tiles = (ns + TILE - 1) / TILE;
    w0 = max(lo / TILE, ns_tiles);
    n_tiles = end > 0 ? ns_tiles + max(0, (end + TILE - 1) / TILE - w0) : 0;
  }
};

// Rows of sequence b in the chunk form; `complain`: report bounds that do not hold.
__device__ __forceinline__ void chunk_rows(const Q8AttnParams &p, int b, bool complain, int &t0, int &nq, int &pos0, int &limit) {
  limit = min(p.max_kv_len, p.c.max_pos);
  const int a = min(max(__ldg(p.r.tok_start + b), 0), p.r.total), e = min(max(__ldg(p.r.tok_start + b + 1), a), p.r.total);
  t0 = a;
  nq = e - a;
  pos0 = __ldg(p.r.start_pos + b);
  if (nq > 0 && complain) {
    const long last = static_cast<long>(pos0) + nq - 1;
    if (pos0 < 0 || last >= p.c.max_pos) report(p.c.error_flag, kStatusOutsideCache);
    else if (last >= limit || nq > p.max_new) report(p.c.error_flag, kStatusLengthBeyondBound);
  }
}

// Share c of a line of W tiles cut for n <= 296 CTAs, and the CTA that owns tile x.  Lines of less than 2^23
// tiles, which is nearly all of them, do without a 64-bit division (some 600 cycles).
__device__ __forceinline__ long share_begin(long W, int n, int c) {
  if (W < (1L << 23)) return static_cast<uint32_t>(c) * static_cast<uint32_t>(W) / static_cast<uint32_t>(n);
  return static_cast<long>(c) * W / n;
}
__device__ __forceinline__ int share_of(long W, int n, long x) {
  if (W < (1L << 23)) return static_cast<int>((static_cast<uint32_t>(x + 1) * static_cast<uint32_t>(n) - 1u) / static_cast<uint32_t>(W));
  return static_cast<int>(((x + 1) * n - 1) / W);
}

} // namespace q8

// Joins pieces [begin, end) of a row: normalised partials o[slot row][128] and log-sum-exps (log2 domain), 32
// pieces a round whose weights the lanes work out together; all 32 lanes, four elements each, pieces in order.
// slot_row(i): where piece i lies.  The result is acc / W at the maximum M; a NaN anywhere makes it NaN.
struct Joined {
  float4 acc;
  float M, W;
};
template <typename F>
__device__ __forceinline__ Joined join_pieces(const float *o, const float *lse, int begin, int end, int lane, F slot_row) {
  Joined r;
  r.M = -INFINITY, r.W = 0.f;
  r.acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = begin; base < end; base += 32) {
    const int n = min(32, end - base);
    const long row = lane < n ? slot_row(base + lane) : 0;
    const float l = lane < n ? __ldcg(lse + row) : -INFINITY;
    float mx = l;
#pragma unroll
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float Mn = fmaxf(r.M, mx), ms = Mn == -INFINITY ? 0.f : Mn;
    const float w = exp2f(l - ms), f = exp2f(r.M - ms);
    r.acc.x *= f, r.acc.y *= f, r.acc.z *= f, r.acc.w *= f;
    r.W *= f;
    r.M = Mn;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      const long ri = __shfl_sync(0xffffffffu, row, i);
      const float4 v = __ldcg(reinterpret_cast<const float4 *>(o + ri * kHeadDim) + lane);
      r.W += wi;
      r.acc.x += wi * v.x, r.acc.y += wi * v.y, r.acc.z += wi * v.z, r.acc.w += wi * v.w;
    }
  }
  return r;
}

// The rows of one cut run: a CTA of eight warps, `split` of them on a row, takes rows blockIdx.y * 8 / split ..
// and so on, gridDim.y CTAs apart.  store(rho, four elements of this lane).
constexpr int kMergeWarps = 8;
template <typename F, typename S>
__device__ __forceinline__ void merge_rows(const float *o, const float *lse, int parts, int rows, int split, F slot_row, S store) {
  __shared__ float4 xo[kMergeWarps][32];
  __shared__ float2 xml[kMergeWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % split, per = kMergeWarps / split;
  for (int r0 = blockIdx.y * per; r0 < rows; r0 += gridDim.y * per) {
    const int rho = r0 + warp / split;
    Joined j;
    j.acc = make_float4(0.f, 0.f, 0.f, 0.f);
    j.M = -INFINITY, j.W = 0.f;
    if (rho < rows)
      j = join_pieces(o, lse, parts * sub / split, parts * (sub + 1) / split, lane, [&](int i) { return slot_row(i, rho); });
    if (split > 1) {
      xo[warp][lane] = j.acc;
      if (lane == 0) xml[warp] = make_float2(j.M, j.W);
      __syncthreads();
      if (sub == 0) {
        float M = -INFINITY;
        for (int x = 0; x < split; ++x) M = fmaxf(M, xml[warp + x].x);
        const float ms = M == -INFINITY ? 0.f : M;
        j.acc = make_float4(0.f, 0.f, 0.f, 0.f), j.W = 0.f;
        for (int x = 0; x < split; ++x) {
          const float2 ml = xml[warp + x];
          if (ml.y == 0.f) continue;     // no piece, or none that sees anything
          const float f = exp2f(ml.x - ms);
          const float4 u = xo[warp + x][lane];
          j.W += f * ml.y;
          j.acc.x += f * u.x, j.acc.y += f * u.y, j.acc.z += f * u.z, j.acc.w += f * u.w;
        }
      }
      __syncthreads();
    }
    if (sub == 0 && rho < rows) {
      if (j.W != 0.f) j.acc.x /= j.W, j.acc.y /= j.W, j.acc.z /= j.W, j.acc.w /= j.W; // NaN divides too
      store(rho, j.acc);
    }
  }
}
// Grid and split of a merge over `runs` runs of `rows` rows, cut for `ctas` CTAs: enough CTAs to fill the GPU,
// few enough that those of runs that were not cut leave soon (ragged prompts, 640 runs: 347 us in all with 512 / runs
// CTAs a run, 305 with 2048, 298 with 4096); several warps on a row where a run can have many pieces (20 tokens of 6
// heads behind 30000 positions, 74 pieces: the call takes 67 us with a warp per row, 31 so).
inline void merge_shape(long runs, int rows, int ctas, dim3 *grid, int *split) {
  *split = ctas >= 16 * runs ? 8 : ctas >= 8 * runs ? 4 : 1;
  const long per = kMergeWarps / *split, most = (rows + per - 1) / per;
  long gy = (4096 + runs - 1) / runs;
  gy = gy > most ? most : gy < 1 ? 1 : gy;
  *grid = dim3(static_cast<unsigned>(runs), static_cast<unsigned>(gy));
}

template <typename... Args>
inline cudaError_t launch_dependent(void (*kernel)(Args...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

} // namespace b200attn
