// C ABI of the 8-bit KV cache operators (declared in include/gpu_ops.h): argument validation on the
// host and dispatch.  No entry point allocates device memory.
#include "gpu_ops.h"
#include "kernels.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>

using namespace b200attn;

namespace {

int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}

int cuda_fail(cudaError_t e, const char *what) { return fail(GPU_OPS_E_CUDA, "%s: %s", what, cudaGetErrorString(e)); }

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The geometry every operator of the set shares.
int check_geometry(const gpu_attn_desc *d) {
  if (!d) return fail(GPU_OPS_E_INVALID, "desc is NULL");
  if (d->dtype != GPU_DT_FLOAT16 && d->dtype != GPU_DT_BFLOAT16)
    return fail(GPU_OPS_E_UNSUPPORTED, "dtype %d: only fp16 (4) and bf16 (5) are supported", d->dtype);
  if (d->head_dim != 128) return fail(GPU_OPS_E_UNSUPPORTED, "head_dim %d: only 128 is supported", d->head_dim);
  if (d->batch <= 0 || d->n_heads <= 0 || d->n_kv_heads <= 0 || d->n_heads % d->n_kv_heads)
    return fail(GPU_OPS_E_INVALID, "batch %d, n_heads %d, n_kv_heads %d", d->batch, d->n_heads, d->n_kv_heads);
  if (d->n_heads > 65535) return fail(GPU_OPS_E_UNSUPPORTED, "n_heads %d: at most 65535", d->n_heads);
  return GPU_OPS_OK;
}

// A row stride of a 16-bit tensor of `heads` heads.
int check_row(const char *what, int64_t stride, int heads) {
  if (stride % 8 || stride < static_cast<int64_t>(heads) * 128)
    return fail(GPU_OPS_E_INVALID, "%s %lld: a multiple of 8 elements, at least %lld", what, static_cast<long long>(stride),
                static_cast<long long>(heads) * 128);
  return GPU_OPS_OK;
}

int cache_from(const gpu_attn_desc *d, const gpu_kv_pages *pages, const gpu_kv_q8 *kv, Q8Cache *c) {
  if (!kv) return fail(GPU_OPS_E_INVALID, "kv is NULL");
  if (!kv->k || !kv->v || !kv->k_exp || !kv->v_exp) return fail(GPU_OPS_E_INVALID, "null cache pointer");
  if (!aligned16(kv->k) || !aligned16(kv->v) || !aligned16(kv->k_exp) || !aligned16(kv->v_exp))
    return fail(GPU_OPS_E_INVALID, "cache pointers must be 16-byte aligned");
  if (kv->max_pos <= 0 || kv->max_pos > (1 << 30)) return fail(GPU_OPS_E_INVALID, "max_pos %d", kv->max_pos);
  *c = Q8Cache{};
  c->k = static_cast<uint8_t *>(kv->k);
  c->v = static_cast<uint8_t *>(kv->v);
  c->kx = kv->k_exp;
  c->vx = kv->v_exp;
  c->c_outer = d->cache_seq_stride;
  c->c_head = d->cache_head_stride;
  c->c_pos = d->cache_pos_stride;
  c->x_outer = kv->exp_outer_stride;
  c->x_head = kv->exp_head_stride;
  c->max_pos = kv->max_pos;
  c->batch = d->batch;
  c->n_kv_heads = d->n_kv_heads;
  long outers = d->batch, rows = kv->max_pos;
  if (pages) {
    if (!pages->page_table) return fail(GPU_OPS_E_INVALID, "null page table");
    const int ps = pages->page_size;
    if (ps < 64 || (ps & (ps - 1))) return fail(GPU_OPS_E_UNSUPPORTED, "page size %d: a power of two >= 64", ps);
    if (pages->table_stride <= 0 || pages->page_stride <= 0 || pages->n_pages <= 0)
      return fail(GPU_OPS_E_INVALID, "table stride %d, page stride %lld, pages %d", pages->table_stride,
                  static_cast<long long>(pages->page_stride), pages->n_pages);
    if (kv->max_pos > static_cast<int64_t>(pages->table_stride) * ps)
      return fail(GPU_OPS_E_INVALID, "max_pos %d: the page table rows hold %lld positions", kv->max_pos,
                  static_cast<long long>(pages->table_stride) * ps);
    c->pg.table = pages->page_table;
    c->pg.page_stride = pages->page_stride;
    c->pg.table_stride = pages->table_stride;
    c->pg.n_pages = pages->n_pages;
    while ((1 << c->pg.page_shift) < ps) ++c->pg.page_shift;
    c->c_outer = pages->page_stride;
    outers = pages->n_pages;
    rows = ps;
  }
  if (c->c_outer % 16 || c->c_head % 16 || c->c_pos % 16 || c->x_outer % 16 || c->x_head % 16)
    return fail(GPU_OPS_E_INVALID, "strides of an 8-bit cache must be multiples of 16 bytes");
  // rows, heads and sequences (pages) may be nested in any order, but must not overlap
  if (c->c_pos < 128 || (d->n_kv_heads > 1 && c->c_head < 128) || (outers > 1 && c->c_outer < 128) || c->c_head < 0 || c->c_outer < 0)
    return fail(GPU_OPS_E_INVALID, "cache strides: outer %ld, head %ld, position %ld", c->c_outer, c->c_head, c->c_pos);
  // (a dimension whose stride is the larger one has to clear what lies inside it)
  const long all_rows = (rows - 1) * c->c_pos + 128, all_heads = (d->n_kv_heads - 1) * c->c_head + 128;
  const bool heads_outside = c->c_head > c->c_pos;
  if (d->n_kv_heads > 1 && (heads_outside ? all_rows > c->c_head : rows > 1 && all_heads > c->c_pos))
    return fail(GPU_OPS_E_INVALID, "%ld positions do not fit the cache (head stride %ld, position stride %ld)", rows, c->c_head, c->c_pos);
  const long widest = c->c_pos > c->c_head ? c->c_pos : c->c_head;
  const long extent = all_rows + (d->n_kv_heads - 1) * c->c_head;
  if (outers > 1 && c->c_outer >= widest && extent > c->c_outer)
    return fail(GPU_OPS_E_INVALID, "%ld positions do not fit the cache (%ld bytes, the next %s begins at %ld)", rows, extent,
                pages ? "page" : "sequence", c->c_outer);
  const long padded = (rows + 15) / 16 * 16;
  if ((d->n_kv_heads > 1 && c->x_head < padded) || (outers > 1 && c->x_outer < padded) || c->x_head < 0 || c->x_outer < 0)
    return fail(GPU_OPS_E_INVALID, "exponent strides: outer %ld, head %ld; rows of %ld bytes", c->x_outer, c->x_head, padded);
  if (outers > 1 && c->x_outer >= c->x_head && padded * d->n_kv_heads > c->x_outer)
    return fail(GPU_OPS_E_INVALID, "exponent rows of %ld heads do not fit %ld bytes", static_cast<long>(d->n_kv_heads), c->x_outer);
  return GPU_OPS_OK;
}

int ragged_from(const int32_t *tok_start, const int32_t *start_pos, int total, Ragged *r) {
  if (!tok_start) return fail(GPU_OPS_E_INVALID, "null tok_start");
  if (total < 0) return fail(GPU_OPS_E_INVALID, "total_tokens %d", total);
  *r = Ragged{tok_start, start_pos, total};
  return GPU_OPS_OK;
}

// The status word lives in mapped host memory, made on a device's first use of the library.
int status_word(Q8Cache *c) {
  c->error_flag = kernel_error_word_dev();
  return c->error_flag ? GPU_OPS_OK : fail(GPU_OPS_E_CUDA, "no status word");
}

int check_attention(const gpu_attn_desc *d, const void *out, const void *q, int max_kv_len, int window, int n_sink) {
  if (!out || !q) return fail(GPU_OPS_E_INVALID, "null tensor pointer");
  if (!aligned16(out) || !aligned16(q)) return fail(GPU_OPS_E_INVALID, "tensor pointers must be 16-byte aligned");
  const int group = d->n_heads / d->n_kv_heads;
  if (group > 16) return fail(GPU_OPS_E_UNSUPPORTED, "group size %d: at most 16 query heads per KV head", group);
  if (max_kv_len <= 0) return fail(GPU_OPS_E_INVALID, "max_kv_len %d", max_kv_len);
  if (window < 0 || n_sink < 0) return fail(GPU_OPS_E_INVALID, "window %d, n_sink %d", window, n_sink);
  return GPU_OPS_OK;
}

int check_workspace(const void *workspace, size_t given, size_t need) {
  if (need && (!workspace || given < need)) return fail(GPU_OPS_E_WORKSPACE, "workspace of %zu bytes given, %zu needed", given, need);
  if (!aligned16(workspace)) return fail(GPU_OPS_E_INVALID, "workspace must be 16-byte aligned");
  return GPU_OPS_OK;
}

// Chunks of up to 16 query rows of a KV head go to the decode kernel, which takes that many at once; the
// tcgen05 kernel pays for 128 at least.  Measured on both: 16 sequences of 4000 to 8000 positions, 40 / 8 heads,
// 3 tokens each: 71 against 123 us; 8 sequences of up to 3000, 16 MHA heads, 16 tokens: 36 against 60.  More rows
// in several walks over the cache do not pay: 6 tokens of the first case 118 against 125 us, 9 tokens 165 against 127.
bool few_rows(int max_new, int group) { return static_cast<long>(max_new) * group <= 16; }

float scale_log2_of_128() { return (1.0f / sqrtf(128.0f)) * 1.4426950408889634f; }

} // namespace

extern "C" {

int gpu_rope_kv_append_q8_layer(const gpu_attn_desc *desc, const gpu_kv_pages *pages, const gpu_kv_q8 *kv, void *q_out,
                                const void *q_in, const void *k_in, const void *v_in, const void *freqs_cis_dev,
                                const int32_t *tok_start_dev, const int32_t *start_pos_dev, int total_tokens,
                                gpu_stream_t stream) {
  if (int rc = check_geometry(desc)) return rc;
  Q8AppendParams p{};
  if (int rc = cache_from(desc, pages, kv, &p.c)) return rc;
  if (int rc = ragged_from(tok_start_dev, start_pos_dev, total_tokens, &p.r)) return rc;
  if (!k_in || !v_in || !freqs_cis_dev || !start_pos_dev || (q_out && !q_in)) return fail(GPU_OPS_E_INVALID, "null tensor pointer");
  if (!aligned16(q_out) || !aligned16(q_in) || !aligned16(k_in) || !aligned16(v_in) || !aligned16(freqs_cis_dev))
    return fail(GPU_OPS_E_INVALID, "tensor pointers must be 16-byte aligned");
  if (q_out)
    if (int rc = check_row("q_tok_stride", desc->q_tok_stride, desc->n_heads)) return rc;
  if (int rc = check_row("kv_in_tok_stride", desc->kv_in_tok_stride, desc->n_kv_heads)) return rc;
  if (total_tokens == 0) return GPU_OPS_OK;
  if (int rc = status_word(&p.c)) return rc;
  p.q_out = q_out;
  p.q = q_in;
  p.k = k_in;
  p.v = v_in;
  p.freqs_cis = static_cast<const float *>(freqs_cis_dev);
  p.q_tok = desc->q_tok_stride;
  p.kv_tok = desc->kv_in_tok_stride;
  p.n_heads = desc->n_heads;
  p.is_neox = desc->is_neox_style ? 1 : 0;
  cudaError_t e = launch_kv_append_q8(p, desc->dtype == GPU_DT_BFLOAT16, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "8-bit rope + append launch");
  add_launch_count(1);
  return GPU_OPS_OK;
}

int gpu_kv_read_q8_layer(const gpu_attn_desc *desc, const gpu_kv_pages *pages, const gpu_kv_q8 *kv, void *k_out, void *v_out,
                         const int32_t *tok_start_dev, const int32_t *start_pos_dev, int total_tokens, gpu_stream_t stream) {
  if (int rc = check_geometry(desc)) return rc;
  Q8ReadParams p{};
  if (int rc = cache_from(desc, pages, kv, &p.c)) return rc;
  if (int rc = ragged_from(tok_start_dev, start_pos_dev, total_tokens, &p.r)) return rc;
  if (!k_out && !v_out) return fail(GPU_OPS_E_INVALID, "no output given");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(GPU_OPS_E_INVALID, "tensor pointers must be 16-byte aligned");
  if (int rc = check_row("kv_in_tok_stride", desc->kv_in_tok_stride, desc->n_kv_heads)) return rc;
  if (total_tokens == 0) return GPU_OPS_OK;
  if (int rc = status_word(&p.c)) return rc;
  p.k_out = k_out;
  p.v_out = v_out;
  p.kv_tok = desc->kv_in_tok_stride;
  cudaError_t e = launch_kv_read_q8(p, desc->dtype == GPU_DT_BFLOAT16, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "8-bit cache read launch");
  add_launch_count(1);
  return GPU_OPS_OK;
}

size_t gpu_attn_decode_q8_workspace_bytes(const gpu_attn_desc *desc, int max_kv_len) {
  if (!desc || desc->batch <= 0 || desc->n_kv_heads <= 0 || desc->n_heads < desc->n_kv_heads || max_kv_len <= 0) return 0;
  return attn_q8_decode_ws_bytes(desc->batch, desc->n_kv_heads, desc->n_heads / desc->n_kv_heads, max_kv_len);
}

int gpu_attn_decode_q8_layer(const gpu_attn_desc *desc, const gpu_kv_pages *pages, const gpu_kv_q8 *kv, void *out, const void *q,
                             const int32_t *kv_len_dev, int max_kv_len, int window, int n_sink, void *workspace,
                             size_t workspace_bytes, gpu_stream_t stream) {
  if (int rc = check_geometry(desc)) return rc;
  Q8AttnParams p{};
  if (int rc = cache_from(desc, pages, kv, &p.c)) return rc;
  if (int rc = check_attention(desc, out, q, max_kv_len, window, n_sink)) return rc;
  if (!kv_len_dev) return fail(GPU_OPS_E_INVALID, "null kv_len");
  if (int rc = check_row("q_seq_stride", desc->q_seq_stride, desc->n_heads)) return rc;
  if (int rc = check_row("out_seq_stride", desc->out_seq_stride, desc->n_heads)) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, gpu_attn_decode_q8_workspace_bytes(desc, max_kv_len))) return rc;
  if (int rc = status_word(&p.c)) return rc;
  p.kv_len = kv_len_dev;
  p.out = out;
  p.q = q;
  p.q_row = desc->q_seq_stride;
  p.out_row = desc->out_seq_stride;
  p.n_heads = desc->n_heads;
  p.group = desc->n_heads / desc->n_kv_heads;
  p.max_kv_len = max_kv_len;
  p.max_new = 1;
  p.window = window;
  p.n_sink = n_sink;
  p.scale_log2 = scale_log2_of_128();
  p.ws = workspace;
  int launches = 0;
  cudaError_t e = launch_attn_q8_decode(p, desc->dtype == GPU_DT_BFLOAT16, static_cast<cudaStream_t>(stream), &launches);
  add_launch_count(launches);
  if (e == cudaErrorNotSupported) return fail(GPU_OPS_E_UNSUPPORTED, "the cache strides cannot be described by a TMA tensor map");
  if (e != cudaSuccess) return cuda_fail(e, "8-bit decode attention launch");
  return GPU_OPS_OK;
}

size_t gpu_attn_chunk_q8_workspace_bytes(const gpu_attn_desc *desc, int total_tokens, int max_new, int max_kv_len) {
  if (!desc || desc->batch <= 0 || desc->n_kv_heads <= 0 || desc->n_heads < desc->n_kv_heads || total_tokens <= 0 || max_new <= 0 ||
      max_kv_len <= 0)
    return 0;
  if (few_rows(max_new, desc->n_heads / desc->n_kv_heads))
    return attn_q8_decode_ws_bytes(desc->batch, desc->n_kv_heads, max_new * (desc->n_heads / desc->n_kv_heads), max_kv_len);
  return attn_q8_chunk_ws_bytes(desc->batch, desc->n_kv_heads, desc->n_heads / desc->n_kv_heads, total_tokens, max_kv_len);
}

int gpu_attn_chunk_q8_layer(const gpu_attn_desc *desc, const gpu_kv_pages *pages, const gpu_kv_q8 *kv, void *out, const void *q,
                            const int32_t *tok_start_dev, const int32_t *start_pos_dev, int total_tokens, int max_new,
                            int max_kv_len, int window, int n_sink, void *workspace, size_t workspace_bytes,
                            gpu_stream_t stream) {
  if (int rc = check_geometry(desc)) return rc;
  Q8AttnParams p{};
  if (int rc = cache_from(desc, pages, kv, &p.c)) return rc;
  if (int rc = ragged_from(tok_start_dev, start_pos_dev, total_tokens, &p.r)) return rc;
  if (int rc = check_attention(desc, out, q, max_kv_len, window, n_sink)) return rc;
  if (!start_pos_dev) return fail(GPU_OPS_E_INVALID, "null start_pos");
  if (max_new <= 0) return fail(GPU_OPS_E_INVALID, "max_new %d", max_new);
  if (int rc = check_row("q_tok_stride", desc->q_tok_stride, desc->n_heads)) return rc;
  if (int rc = check_row("out_tok_stride", desc->out_tok_stride, desc->n_heads)) return rc;
  if (!few_rows(max_new, desc->n_heads / desc->n_kv_heads) && desc->batch > kChunkMaxBatch)
    return fail(GPU_OPS_E_UNSUPPORTED, "batch %d: at most %d sequences", desc->batch, kChunkMaxBatch);
  if (total_tokens == 0) return GPU_OPS_OK;
  if (int rc = check_workspace(workspace, workspace_bytes, gpu_attn_chunk_q8_workspace_bytes(desc, total_tokens, max_new, max_kv_len)))
    return rc;
  if (int rc = status_word(&p.c)) return rc;
  p.out = out;
  p.q = q;
  p.q_row = desc->q_tok_stride;
  p.out_row = desc->out_tok_stride;
  p.n_heads = desc->n_heads;
  p.group = desc->n_heads / desc->n_kv_heads;
  p.max_kv_len = max_kv_len;
  p.max_new = max_new;
  p.window = window;
  p.n_sink = n_sink;
  p.scale_log2 = scale_log2_of_128();
  p.ws = workspace;
  int launches = 0;
  const bool bf16 = desc->dtype == GPU_DT_BFLOAT16;
  cudaError_t e = few_rows(max_new, p.group) ? launch_attn_q8_decode(p, bf16, static_cast<cudaStream_t>(stream), &launches)
                                             : launch_attn_q8_chunk(p, bf16, static_cast<cudaStream_t>(stream), &launches);
  add_launch_count(launches);
  if (e == cudaErrorNotSupported) return fail(GPU_OPS_E_UNSUPPORTED, "the cache strides cannot be described by a TMA tensor map");
  if (e != cudaSuccess) return cuda_fail(e, "8-bit chunk attention launch");
  return GPU_OPS_OK;
}

} // extern "C"
