// Attention over the 8-bit KV cache, plain form: one CTA per (query row, head), four warps that take
// every fourth visible position.  A lane holds four of the 128 elements; a position's score is one warp
// reduction, and its weight joins a running maximum and sum, so the cache is read once.
#include "q8.cuh"

namespace b200attn {

namespace {

using namespace q8;

__device__ __forceinline__ float4 codes4(uint32_t w) {
  const float2 a = Elem<__half>::unpack(cvt_e4m3x2_f16x2(w & 0xffffu)), b = Elem<__half>::unpack(cvt_e4m3x2_f16x2(w >> 16));
  return make_float4(a.x, a.y, b.x, b.y);
}

template <typename T> __global__ void __launch_bounds__(128) attn_q8_kernel(Q8AttnParams p) {
  __shared__ float4 xo[4][32];
  __shared__ float2 xml[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, kvh = h / p.group;
  const int t = blockIdx.x;
  int b, pos;
  if (p.kv_len) {
    b = t;
    int len = max(0, __ldg(p.kv_len + b));
    if (len > min(p.max_kv_len, p.c.max_pos)) {
      report(p.c.error_flag, kStatusLengthBeyondBound);
      len = min(p.max_kv_len, p.c.max_pos);
    }
    pos = len - 1;
  } else {
    b = seq_of_row(p.r.tok_start, p.c.batch, t, lane);
    if (b >= p.c.batch) return;
    const int r = t - __ldg(p.r.tok_start + b);
    if (r < 0) return;
    pos = __ldg(p.r.start_pos + b) + r;
    if (pos >= p.c.max_pos) {
      report(p.c.error_flag, kStatusOutsideCache);
      pos = p.c.max_pos - 1;
    } else if (pos >= p.max_kv_len) {
      report(p.c.error_flag, kStatusLengthBeyondBound);
      pos = p.max_kv_len - 1;
    }
  }
  const T *qrow = static_cast<const T *>(p.q) + static_cast<long>(t) * p.q_row + h * kHeadDim + 4 * lane;
  const uint2 qu = *reinterpret_cast<const uint2 *>(qrow);
  const float2 q01 = Elem<T>::unpack(qu.x), q23 = Elem<T>::unpack(qu.y);
  const int lo = window_begin(pos, p.window), n_sink = min(p.n_sink, lo);
  float M = -INFINITY, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = warp; i < n_sink + pos + 1 - lo; i += 4) {
    const int j = i < n_sink ? i : lo + i - n_sink;
    long outer;
    int in_pos;
    if (!locate(p.c, b, j, outer, in_pos)) {
      report(p.c.error_flag, kStatusOutsideCache);
      outer = 0, in_pos = 0;
    }
    const long co = outer * p.c.c_outer + kvh * p.c.c_head + static_cast<long>(in_pos) * p.c.c_pos + 4 * lane;
    const long xo_ = outer * p.c.x_outer + kvh * p.c.x_head + in_pos;
    const float4 k = codes4(*reinterpret_cast<const uint32_t *>(p.c.k + co));
    const float4 v = codes4(*reinterpret_cast<const uint32_t *>(p.c.v + co));
    const int kx = p.c.kx[xo_], vx = p.c.vx[xo_];
    float s = q01.x * k.x + q01.y * k.y + q23.x * k.z + q23.y * k.w;
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= p.scale_log2 * pow2i(kx - 127);
    if (kx == kPoison || vx == kPoison) s = __int_as_float(0x7fc00000);
    const float mn = fmaxf(M, s);
    const float f = exp2f(M - mn), w = exp2f(s - mn);
    const float wv = w * pow2i(vx - 127);
    L = L * f + w;
    o.x = o.x * f + wv * v.x, o.y = o.y * f + wv * v.y, o.z = o.z * f + wv * v.z, o.w = o.w * f + wv * v.w;
    M = mn;
  }
  xo[warp][lane] = o;
  if (lane == 0) xml[warp] = make_float2(M, L);
  __syncthreads();
  if (warp != 0) return;
  float Mx = fmaxf(fmaxf(xml[0].x, xml[1].x), fmaxf(xml[2].x, xml[3].x));
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float W = 0.f;
  for (int x = 0; x < 4; ++x) {
    if (xml[x].x == -INFINITY && xml[x].y == 0.f) continue;
    const float f = exp2f(xml[x].x - Mx);
    W += f * xml[x].y;
    a.x += f * xo[x][lane].x, a.y += f * xo[x][lane].y, a.z += f * xo[x][lane].z, a.w += f * xo[x][lane].w;
  }
  if (W != 0.f) a.x /= W, a.y /= W, a.z /= W, a.w /= W; // NaN divides too
  uint2 u;
  u.x = Elem<T>::pack(a.x, a.y);
  u.y = Elem<T>::pack(a.z, a.w);
  *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + static_cast<long>(t) * p.out_row + h * kHeadDim + 4 * lane) = u;
}

} // namespace

cudaError_t launch_attn_q8(const Q8AttnParams &p, bool bf16, cudaStream_t stream, int *launches) {
  const dim3 grid(p.kv_len ? p.c.batch : p.r.total, p.n_heads);
  if (bf16) attn_q8_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(p);
  else attn_q8_kernel<__half><<<grid, 128, 0, stream>>>(p);
  *launches = 1;
  return cudaGetLastError();
}

} // namespace b200attn
