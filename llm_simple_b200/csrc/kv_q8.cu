// Writing the 8-bit KV cache (RoPE + quantise + append of a ragged batch) and reading rows of it back
// to 16 bits.
//
// Eight threads work on one row of 128 elements (a token and a head), sixteen elements each, so that
// the row's largest magnitude is three shuffles away and its quantised form leaves in one pass: the
// row is read once and written once.  Both kernels are bound by HBM: 256 B in and 129 B out per
// written row (256 B out for a query row), 129 B in and 256 B out per row read back.
#include "q8.cuh"

namespace b200attn {

namespace {

using namespace q8;

constexpr int kThreads = 256;
// CTAs per SM and rows of a thread group under way in the read kernel.  More CTAs are slower: many streams of
// reads and writes at once cost HBM more than they hide (137,000 positions of 8 KV heads: 147 us with 3 CTAs
// and 4 rows, 151 with 4 and 2, 171 with 6 and 2, 193 with 8 and 2).  The append kernel's values want 64 registers.
constexpr int kAppendCtas = 4, kReadCtas = 3, kAtOnce = 4;
// log2 of the thread groups that share a token in calls of many tokens.  A warp of the read kernel takes four
// neighbouring positions of a head, 512 contiguous bytes of codes (eight groups per token: 180 us); the append
// kernel reads mostly Q, whose heads are neighbours (prompts of 37 to 3900 tokens: 171 us with 0, 166 with 2).
constexpr int kAppendLanes = 2, kReadLanes = 0;

// Rotates the pairs of two 8-element chunks in fp32: chunks (2i, 2i + 1) for the interleaved pairing,
// (i, i + 8) for the neox pairing.  Same products and sums as rope_pair everywhere else, no rounding
// to 16 bits.
__device__ __forceinline__ void rotate16(float (&x)[16], const float4 *tab, bool neox) {
#pragma unroll
  for (int f = 0; f < 8; ++f) {
    const float4 cs = tab[f >> 1];
    const float c = (f & 1) ? cs.z : cs.x, s = (f & 1) ? cs.w : cs.y;
    float a, b;
    if (neox) {
      rope_pair(x[f], x[8 + f], c, s, a, b);
      x[f] = a, x[8 + f] = b;
    } else {
      rope_pair(x[2 * f], x[2 * f + 1], c, s, a, b);
      x[2 * f] = a, x[2 * f + 1] = b;
    }
  }
}

template <typename T> __device__ __forceinline__ void unpack16(const uint4 &u0, const uint4 &u1, float (&x)[16]) {
  const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = Elem<T>::unpack(w[i]);
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}

template <typename T> __device__ __forceinline__ uint4 pack8(const float *x) {
  return make_uint4(Elem<T>::pack(x[0], x[1]), Elem<T>::pack(x[2], x[3]), Elem<T>::pack(x[4], x[5]), Elem<T>::pack(x[6], x[7]));
}

// A group of eight threads stays with one token and walks its head rows `lanes` apart, as in
// rope_append_kernel: the thread's share of the table row and the token's place are fetched once.
template <typename T> __global__ void __launch_bounds__(kThreads, kAppendCtas) kv_append_q8_kernel(Q8AppendParams p, int lanes_log2) {
  const int i = threadIdx.x & 7, lane = threadIdx.x & 31;
  const int grp = threadIdx.x >> 3;
  const int lanes = 1 << lanes_log2;
  const int t = blockIdx.x * (32 >> lanes_log2) + (grp >> lanes_log2);
  const int b = seq_of_row(p.r.tok_start, p.c.batch, min(t, p.r.total - 1), lane);
  const int r = b < p.c.batch ? t - __ldg(p.r.tok_start + b) : -1;
  const bool live = t < p.r.total && r >= 0;
  const int pos = live ? __ldg(p.r.start_pos + b) + r : -1;
  long outer = 0;
  int in_pos = 0;
  const bool table_ok = live && static_cast<unsigned>(pos) < static_cast<unsigned>(p.c.max_pos); // the RoPE row exists
  const bool stored = table_ok && locate(p.c, b, pos, outer, in_pos);
  if (live && !stored && i == 0) report(p.c.error_flag, kStatusOutsideCache);
  float4 tab[4];
  if (table_ok) {
    const float4 *row = reinterpret_cast<const float4 *>(p.freqs_cis + static_cast<long>(pos) * kHeadDim + 16 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) tab[e] = __ldg(row + e);
  }
  const int hq = p.q_out ? p.n_heads : 0, hk = p.c.n_kv_heads;
  const int slots = hq + 2 * hk;
  const int step = lanes * gridDim.z;
  auto kind = [&](int slot) { return slot < hq ? 0 : slot < hq + hk ? 1 : 2; };                       // q, k, v
  auto wanted = [&](int slot) { return slot < slots && (kind(slot) == 0 ? table_ok : stored); };
  // The next row is requested before this one is worked on: a thread's 32 bytes at a time do not cover
  // the latency of HBM.
  uint4 n0 = make_uint4(0, 0, 0, 0), n1 = n0;
  auto request = [&](int slot) {
    if (!wanted(slot)) return;
    const int which = kind(slot), h = slot - (which == 0 ? 0 : which == 1 ? hq : hq + hk);
    const bool split = which < 2 && p.is_neox; // the thread's two chunks are 64 elements apart
    const T *src = static_cast<const T *>(which == 0 ? p.q : which == 1 ? p.k : p.v) +
                   static_cast<long>(t) * (which == 0 ? p.q_tok : p.kv_tok) + h * kHeadDim;
    n0 = __ldcs(reinterpret_cast<const uint4 *>(src + (split ? i : 2 * i) * 8));
    n1 = __ldcs(reinterpret_cast<const uint4 *>(src + (split ? i + 8 : 2 * i + 1) * 8));
  };
  const int slot0 = blockIdx.z * lanes + (grp & (lanes - 1));
  request(slot0);
  for (int slot = slot0; slot - (grp & (lanes - 1)) < slots; slot += step) { // the same rounds for all lanes of a warp
    const int which = kind(slot);
    const bool on = wanted(slot);
    const bool rotated = which < 2;
    const bool split = rotated && p.is_neox;
    const int c0 = split ? i : 2 * i, c1 = split ? i + 8 : 2 * i + 1;
    const int h = slot - (which == 0 ? 0 : which == 1 ? hq : hq + hk);
    float x[16];
    const uint4 u0 = n0, u1 = n1;
    request(slot + step);
    if (on) {
      unpack16<T>(u0, u1, x);
      if (rotated) rotate16(x, tab, p.is_neox != 0);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = 0.f;
    }
    // largest bit pattern of |x| over the row: infinities and NaN compare above every finite value
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!on) continue;
    if (which == 0) {
      T *dst = static_cast<T *>(p.q_out) + static_cast<long>(t) * p.q_tok + h * kHeadDim;
      *reinterpret_cast<uint4 *>(dst + c0 * 8) = pack8<T>(x);
      *reinterpret_cast<uint4 *>(dst + c1 * 8) = pack8<T>(x + 8);
      continue;
    }
    const bool poison = top >= 0x7f800000u;
    const int e = poison ? 0 : row_exp(__uint_as_float(top));
    const float inv = pow2i(-e); // exact: e lies in -100 .. 120
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = poison ? 0u : cvt_f32_e4m3x2(x[4 * j] * inv, x[4 * j + 1] * inv) |
                               (cvt_f32_e4m3x2(x[4 * j + 2] * inv, x[4 * j + 3] * inv) << 16);
    }
    uint8_t *dst = (which == 1 ? p.c.k : p.c.v) + outer * p.c.c_outer + h * p.c.c_head + static_cast<long>(in_pos) * p.c.c_pos;
    *reinterpret_cast<uint2 *>(dst + c0 * 8) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2 *>(dst + c1 * 8) = make_uint2(w[2], w[3]);
    if (i == 0)
      ((which == 1 ? p.c.kx : p.c.vx))[outer * p.c.x_outer + h * p.c.x_head + in_pos] = static_cast<uint8_t>(poison ? kPoison : e + 127);
  }
}

template <typename T> __global__ void __launch_bounds__(kThreads, kReadCtas) kv_read_q8_kernel(Q8ReadParams p, int lanes_log2) {
  const int i = threadIdx.x & 7, lane = threadIdx.x & 31;
  const int grp = threadIdx.x >> 3;
  const int lanes = 1 << lanes_log2;
  const int t = blockIdx.x * (32 >> lanes_log2) + (grp >> lanes_log2);
  const int b = seq_of_row(p.r.tok_start, p.c.batch, min(t, p.r.total - 1), lane);
  if (t >= p.r.total || b >= p.c.batch) return;
  const int r = t - __ldg(p.r.tok_start + b);
  if (r < 0) return;
  const int pos = (p.r.start_pos ? __ldg(p.r.start_pos + b) : 0) + r;
  long outer;
  int in_pos;
  if (!locate(p.c, b, pos, outer, in_pos)) {
    if (i == 0) report(p.c.error_flag, kStatusOutsideCache);
    return;
  }
  const int hk = p.c.n_kv_heads, step = lanes * gridDim.z;
  // several rows are under way at once: 16 bytes a thread do not cover the latency of HBM
  for (int slot = (grp & (lanes - 1)) + blockIdx.z * lanes; slot < 2 * hk; slot += kAtOnce * step) {
    uint4 u[kAtOnce];
    int x[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int s = slot + k * step;
      const bool is_v = s >= hk;
      if (s >= 2 * hk || !(is_v ? p.v_out : p.k_out)) continue;
      const int h = s - (is_v ? hk : 0);
      u[k] = __ldcs(reinterpret_cast<const uint4 *>((is_v ? p.c.v : p.c.k) + outer * p.c.c_outer + h * p.c.c_head +
                                                    static_cast<long>(in_pos) * p.c.c_pos + 16 * i));
      x[k] = (is_v ? p.c.vx : p.c.kx)[outer * p.c.x_outer + h * p.c.x_head + in_pos];
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int s = slot + k * step;
      const bool is_v = s >= hk;
      T *out = static_cast<T *>(is_v ? p.v_out : p.k_out);
      if (s >= 2 * hk || !out) continue;
      const float f = x[k] == kPoison ? __int_as_float(0x7fc00000) : x[k] > 0 ? pow2i(x[k] - 127) : 0.f;
      const uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
      uint32_t o[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t lo, hi;
        cvt_e4m3x4_f16x4(w[j], lo, hi);
        const float2 a = Elem<__half>::unpack(lo), b2 = Elem<__half>::unpack(hi);
        o[2 * j] = Elem<T>::pack(a.x * f, a.y * f);
        o[2 * j + 1] = Elem<T>::pack(b2.x * f, b2.y * f);
      }
      T *dst = out + static_cast<long>(t) * p.kv_tok + (s - (is_v ? hk : 0)) * kHeadDim + 16 * i;
      __stcs(reinterpret_cast<uint4 *>(dst), make_uint4(o[0], o[1], o[2], o[3]));
      __stcs(reinterpret_cast<uint4 *>(dst) + 1, make_uint4(o[4], o[5], o[6], o[7]));
    }
  }
}

// Thread groups per token, 2^l at least: calls of few tokens spread a token's head rows over more groups,
// and over CTAs, so that they still fill the GPU.
void shape_of(long tokens, int slots, int l, int *lanes_log2, dim3 *grid) {
  while (l < 5 && (tokens + (32 >> l) - 1) / (32 >> l) < 148L * 8) ++l;
  while (l > 0 && (1 << (l - 1)) >= slots) --l;
  const int toks = 32 >> l;
  const unsigned gx = static_cast<unsigned>((tokens + toks - 1) / toks);
  unsigned gz = 1;
  if (l == 5 && gx < 148u * 8) gz = static_cast<unsigned>((slots + 31) / 32);
  *lanes_log2 = l;
  *grid = dim3(gx, 1, gz);
}

} // namespace

cudaError_t launch_kv_append_q8(const Q8AppendParams &p, bool bf16, cudaStream_t stream) {
  int l;
  dim3 grid;
  shape_of(p.r.total, (p.q_out ? p.n_heads : 0) + 2 * p.c.n_kv_heads, kAppendLanes, &l, &grid);
  if (bf16) kv_append_q8_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p, l);
  else kv_append_q8_kernel<__half><<<grid, kThreads, 0, stream>>>(p, l);
  return cudaGetLastError();
}

cudaError_t launch_kv_read_q8(const Q8ReadParams &p, bool bf16, cudaStream_t stream) {
  int l;
  dim3 grid;
  shape_of(p.r.total, 2 * p.c.n_kv_heads, kReadLanes, &l, &grid);
  if (bf16) kv_read_q8_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p, l);
  else kv_read_q8_kernel<__half><<<grid, kThreads, 0, stream>>>(p, l);
  return cudaGetLastError();
}

} // namespace b200attn
