// The entry points of a decoder's serving step and of its prompts (declared in include/odla_b200.h): their arguments are checked here, completely,
// before anything is enqueued; the kernels check what only they can see (slots, page numbers, lengths).
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "common.h"

using namespace b200;

namespace {

const int kStorage[3] = {DT_F32, DT_F16, DT_BF16};

bool have_device(const char* what) {
  if (visible_devices() > 0) return true;
  fprintf(stderr, "[odla_b200] %s: no CUDA device (there is no CPU fallback)\n", what);
  return false;
}
struct Extent { long long n, stride; };
// Strides of one tensor: none negative or above 2^46, and no row 2^60 elements or more behind the first, so that offsets stay inside 63 bits.
bool strides_ok(std::initializer_list<Extent> extents) {
  __int128 reach = 0;
  for (const Extent& e : extents) {
    if (e.stride < 0 || e.stride > (1ll << 46)) return false;
    if (e.n > 1) reach += (__int128)(e.n - 1) * e.stride;
  }
  return reach < ((__int128)1 << 60);
}
// Rows that are written must not lie on one another: sorted by stride, each extent above 1 steps over all that the smaller strides reach.  Every dense
// tensor, in any order of its extents, and every slice of one is laid out like that.
bool apart(int channels, std::initializer_list<Extent> extents) {
  Extent sorted[3];
  int n = 0;
  for (const Extent& e : extents)
    if (e.n > 1) sorted[n++] = e;
  std::sort(sorted, sorted + n, [](const Extent& a, const Extent& b) { return a.stride < b.stride; });
  __int128 reach = channels;
  for (int i = 0; i < n; ++i) {
    if (sorted[i].stride < reach) return false;
    reach += (__int128)(sorted[i].n - 1) * sorted[i].stride;
  }
  return true;
}
struct Step { long long extent, from, to; };
// In place: a result's rows lie where the input's do (an extent of one has no step).
bool same_rows(std::initializer_list<Step> steps) {
  for (const Step& s : steps)
    if (s.extent > 1 && s.from != s.to) return false;
  return true;
}
bool element_aligned(int dtype, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p % (dtype == 0 ? 4 : 2)) return false;
  return true;
}
bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p % 16) return false;
  return true;
}

// 1 / (2 pi) as a binary fraction, the first bits first.
constexpr uint64_t kTurnsOfRadian[20] = {
  0x28BE60DB9391054A, 0x7F09D5F47D4D3770, 0x36D8A5664F10E410, 0x7F9458EAF7AEF158, 0x6DC91B8E909374B8,
  0x01924BBA82746487, 0x3F877AC72C4A69CF, 0xBA208D7D4BAED121, 0x3A671C09AD17DF90, 0x4E64758E60D4CE7D,
  0x272117E2EF7E4A0E, 0xC7FE25FFF7816603, 0xFBCBC462D6829B47, 0xDB4D9FB3C9F2C26D, 0xD3D18FD9A797FA8B,
  0x5D49EEB1FAF97C5E, 0xCF41CE7DE294A4BA, 0x9AFED7EC47E35742, 0x1580CC11BF1EDAEA, 0xFC33EF0826BD0D87};
// Turns per position in units of 2^-64, modulo one turn, to the nearest; any finite frequency, of either sign.  The frequency is a whole number of 53
// bits times 2^e, and of 2^e / (2 pi) only the bits behind the point matter: 192 of them are multiplied (M. H. Payne and R. N. Hanek, "Radian reduction
// for trigonometric functions", 1983).
uint64_t turn_units(double radians) {
  uint64_t bits;
  memcpy(&bits, &radians, 8);
  const int field = (int)(bits >> 52 & 0x7ff), e = (field ? field : 1) - 1075;
  const uint64_t m = (bits & ((1ull << 52) - 1)) | (field ? 1ull << 52 : 0);
  auto word = [](int at) -> uint64_t {   // 64 bits from place `at` on; there is nothing in front of the point
    if (at < 0) return at > -64 ? kTurnsOfRadian[0] >> -at : 0;
    const int i = at / 64, s = at % 64;
    return s ? kTurnsOfRadian[i] << s | kTurnsOfRadian[i + 1] >> (64 - s) : kTurnsOfRadian[i];
  };
  typedef unsigned __int128 Wide;
  const Wide low = (Wide)m * word(e + 64) + (uint64_t)((Wide)m * word(e + 128) >> 64);
  const uint64_t u = m * word(e) + (uint64_t)(low >> 64) + (uint64_t)((uint64_t)low >> 63);
  return bits >> 63 ? 0 - u : u;
}
bool spec_ok(const odla_b200_rotary_spec* s, int channels) {
  if (s->pairs < 0 || s->pairs > ODLA_B200_MAX_ROTARY_PAIRS || 2 * s->pairs > channels || s->axes < 1 || s->axes > 4) return false;
  for (int i = 0; i < s->pairs; ++i)
    if (s->axis[i] >= s->axes || !std::isfinite(s->frequency[i])) return false;
  return true;
}
void put_spec(TurnGeom& g, const odla_b200_rotary_spec* s) {
  g.pairs = s ? s->pairs : 0;
  g.interleaved = s && s->interleaved;
  for (int i = 0; i < g.pairs; ++i) { g.frequency[i] = turn_units(s->frequency[i]); g.axis[i] = s->axis[i]; }
}
bool cache_ok(const odla_b200_paged_cache* c) {
  return c && c->dtype >= 0 && c->dtype <= 2 && c->pages >= 1 && c->page_size >= 1 && c->heads >= 1 && c->heads <= 1024 && c->channels >= 1 && c->channels <= 1024 &&
         strides_ok({{c->pages, c->page}, {c->heads, c->head}, {c->page_size, c->token}});
}

bool attention_args(const odla_b200_paged_cache* c, const odla_b200_paged_attention_desc* d, PagedAttention& a) {
  if (!cache_ok(c) || !d || c->dtype == 0 || (c->channels != 64 && c->channels != 128)) return false;
  if (d->batch < 0 || d->queries < 1 || d->heads < 1 || d->heads > 1024 || d->heads % c->heads || d->prefix_length < 0 || d->table_width < 0 || !std::isfinite(d->scale)) return false;
  if (!strides_ok({{d->batch, d->q_batch}, {d->queries, d->q_token}, {d->heads, d->q_head}}) || !strides_ok({{d->batch, d->y_batch}, {d->queries, d->y_token}, {d->heads, d->y_head}}))
    return false;
  if (!apart(c->channels, {{d->batch, d->y_batch}, {d->queries, d->y_token}, {d->heads, d->y_head}})) return false;
  for (long long s : {c->page, c->head, c->token, d->q_batch, d->q_token, d->q_head, d->y_batch, d->y_token, d->y_head})
    if (s % 8) return false;
  // positions are counted in 32 bits, rows of the workspace too
  if ((long long)d->table_width * c->page_size + d->prefix_length >= (1ll << 30)) return false;
  // (two factors first: three ints may pass 64 bits)
  if ((long long)d->batch * d->queries >= (1ll << 24) || (long long)d->batch * d->queries * d->heads >= (1ll << 24)) return false;
  a = PagedAttention{kStorage[c->dtype], d->batch, d->queries, d->heads, c->heads, c->channels, c->pages, c->page_size, d->prefix_length, d->table_width, d->scale,
                     c->page, c->head, c->token, d->q_batch, d->q_token, d->q_head, d->y_batch, d->y_token, d->y_head};
  return true;
}

}  // namespace

extern "C" int odla_b200_rotary(const odla_b200_rotary_spec* spec, const odla_b200_rotary_desc* d, const void* x, void* y, const int* positions, void* stream) {
  if (!spec || !d || d->dtype < 0 || d->dtype > 2 || d->batch < 0 || d->tokens < 0 || d->heads < 0 || d->heads > 1024 || d->channels < 1 || d->channels > 1024) return -1;
  if (!spec_ok(spec, d->channels) || (long long)d->batch * d->tokens >= (1ll << 31)) return -1;
  if (!strides_ok({{d->batch, d->x_batch}, {d->tokens, d->x_token}, {d->heads, d->x_head}}) || !strides_ok({{d->batch, d->y_batch}, {d->tokens, d->y_token}, {d->heads, d->y_head}}))
    return -1;
  if (d->batch == 0 || d->tokens == 0 || d->heads == 0) return 0;
  if (!apart(d->channels, {{d->batch, d->y_batch}, {d->tokens, d->y_token}, {d->heads, d->y_head}})) return -1;
  if (!x || !y || (spec->pairs && !positions) || !element_aligned(d->dtype, {x, y}) || (uintptr_t)positions % 4) return -1;
  if (x == y && !same_rows({{d->batch, d->x_batch, d->y_batch}, {d->tokens, d->x_token, d->y_token}, {d->heads, d->x_head, d->y_head}})) return -1;
  if (!have_device("odla_b200_rotary")) return -2;
  TurnGeom g{};
  g.src[0] = x; g.dst[0] = y;
  g.s_batch = d->x_batch; g.s_token[0] = d->x_token; g.s_head[0] = d->x_head;
  g.d_batch = d->y_batch; g.d_token = d->y_token; g.d_head = d->y_head;
  g.batch = d->batch; g.tokens = d->tokens; g.heads = d->heads; g.channels = d->channels;
  g.heads_outside = d->x_head > d->x_token;
  g.positions = positions;
  put_spec(g, spec);
  return turn_rows(g, kStorage[d->dtype], (cudaStream_t)stream);
}

extern "C" int odla_b200_paged_append(const odla_b200_paged_cache* c, void* key_cache, void* value_cache, const odla_b200_append_desc* d, const odla_b200_rotary_spec* spec,
                                      const void* q, const void* k, const void* v, void* q_out, const int* positions, const long long* slots, void* stream) {
  if (!cache_ok(c) || !d || d->tokens < 0 || d->heads < 0 || d->heads > 1024 || (spec && !spec_ok(spec, c->channels))) return -1;
  if (!strides_ok({{d->tokens, d->q_token}, {d->heads, d->q_head}}) || !strides_ok({{d->tokens, d->k_token}, {c->heads, d->k_head}}) ||
      !strides_ok({{d->tokens, d->v_token}, {c->heads, d->v_head}}) || !strides_ok({{d->tokens, d->y_token}, {d->heads, d->y_head}}))
    return -1;
  if (d->tokens == 0) return 0;
  if (!apart(c->channels, {{c->pages, c->page}, {c->page_size, c->token}, {c->heads, c->head}})) return -1;
  if (d->heads && !apart(c->channels, {{d->tokens, d->y_token}, {d->heads, d->y_head}})) return -1;
  if (!key_cache || !value_cache || !k || !v || !slots || (d->heads && (!q || !q_out)) || (spec && spec->pairs && !positions)) return -1;
  if (!element_aligned(c->dtype, {key_cache, value_cache, q, k, v, q_out}) || (uintptr_t)positions % 4 || (uintptr_t)slots % 8) return -1;
  if (d->heads && q == q_out && !same_rows({{d->tokens, d->q_token, d->y_token}, {d->heads, d->q_head, d->y_head}})) return -1;
  if (!have_device("odla_b200_paged_append")) return -2;
  TurnGeom g{};
  g.src[0] = q; g.src[1] = k; g.src[2] = v;
  g.dst[0] = q_out; g.dst[1] = key_cache; g.dst[2] = value_cache;
  g.s_token[0] = d->q_token; g.s_token[1] = d->k_token; g.s_token[2] = d->v_token;
  g.s_head[0] = d->q_head; g.s_head[1] = d->k_head; g.s_head[2] = d->v_head;
  g.d_token = d->y_token; g.d_head = d->y_head;
  g.c_page = c->page; g.c_token = c->token; g.c_head = c->head;
  g.batch = 1; g.tokens = d->tokens; g.heads = d->heads; g.kv_heads = c->heads; g.channels = c->channels;
  g.pages = c->pages; g.page_size = c->page_size;
  g.positions = positions; g.slots = slots;
  put_spec(g, spec);
  return turn_rows(g, kStorage[c->dtype], (cudaStream_t)stream);
}

extern "C" long long odla_b200_paged_attention_workspace(const odla_b200_paged_cache* c, const odla_b200_paged_attention_desc* d) {
  PagedAttention a;
  return attention_args(c, d, a) ? paged_attention_workspace(a) : -1;
}
extern "C" int odla_b200_paged_attention(const odla_b200_paged_cache* c, const void* key_cache, const void* value_cache, const odla_b200_paged_attention_desc* d, const void* q,
                                         const int* prefix_pages, const int* page_table, const int* lengths, void* y, void* workspace, long long workspace_bytes, void* stream) {
  PagedAttention a;
  if (!attention_args(c, d, a)) return -1;
  if (d->batch == 0) return 0;
  if (!key_cache || !value_cache || !q || !y || !lengths || (d->prefix_length && !prefix_pages) || (d->table_width && !page_table)) return -1;
  if (!aligned16({key_cache, value_cache, q, y, workspace}) || (uintptr_t)prefix_pages % 4 || (uintptr_t)page_table % 4 || (uintptr_t)lengths % 4) return -1;
  const long long need = paged_attention_workspace(a);
  if (need < 0 || workspace_bytes < need || (need && !workspace)) return -1;
  if (!have_device("odla_b200_paged_attention")) return -2;
  return paged_attention(a, key_cache, value_cache, q, prefix_pages, page_table, lengths, y, workspace, (cudaStream_t)stream);
}

extern "C" int odla_b200_sample(const odla_b200_sample_desc* d, const void* logits, const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                                const float* uniform, int* tokens, void* stream) {
  if (!d || d->dtype < 0 || d->dtype > 2 || d->rows < 0 || d->rows > (1 << 24) || d->vocab < 1 || d->vocab > kMaxVocab || !strides_ok({{d->rows, d->row}})) return -1;
  if (d->rows == 0) return 0;
  if (!logits || !uniform || !tokens || !element_aligned(d->dtype, {logits})) return -1;
  for (const void* p : {(const void*)temperature, (const void*)top_k, (const void*)top_p, (const void*)min_p, (const void*)uniform, (const void*)tokens})
    if ((uintptr_t)p % 4) return -1;
  if (!have_device("odla_b200_sample")) return -2;
  return sample(kStorage[d->dtype], d->rows, d->vocab, d->row, logits, temperature, top_k, top_p, min_p, uniform, tokens, (cudaStream_t)stream);
}

extern "C" int odla_b200_rms_norm(const odla_b200_rms_norm_desc* d, const void* x, const void* residual, const void* weight, void* sum, void* y, void* quantised, float* scales,
                                  void* stream) {
  if (!d || d->dtype < 0 || d->dtype > 2 || d->weight_dtype < 0 || d->weight_dtype > 2 || d->rows < 0 || d->heads < 0 || d->heads > 1024 || d->channels < 1 || d->channels > 32768) return -1;
  if (d->quant < 0 || d->quant > 2 || d->group < 0 || !(d->epsilon >= 0.f) || !std::isfinite(d->epsilon) || !std::isfinite(d->weight_offset) || (long long)d->rows * d->heads >= (1ll << 31)) return -1;
  if (d->quant && d->group && (d->channels % d->group || (d->group % 8 && d->group != d->channels))) return -1;
  const long long steps[5][2] = {{d->x_row, d->x_head}, {d->residual_row, d->residual_head}, {d->sum_row, d->sum_head}, {d->y_row, d->y_head}, {d->quant_row, d->quant_head}};
  void* const out[3] = {sum, y, d->quant ? quantised : nullptr};
  const void* const in[2] = {x, residual};
  for (int i = 0; i < 5; ++i)
    if ((i < 2 ? in[i] || i == 0 : out[i - 2] != nullptr) && !strides_ok({{d->rows, steps[i][0]}, {d->heads, steps[i][1]}})) return -1;
  if (d->rows == 0 || d->heads == 0) return 0;
  for (int i = 0; i < 3; ++i)
    if (out[i] && !apart(d->channels, {{d->rows, steps[i + 2][0]}, {d->heads, steps[i + 2][1]}})) return -1;
  if (!x || (sum && !residual) || (!sum && !y && !d->quant) || (d->quant && (!quantised || !scales)) || (!d->quant && quantised)) return -1;
  if (!element_aligned(d->dtype, {x, residual, sum, y}) || !element_aligned(d->weight_dtype, {weight}) || (uintptr_t)scales % 4) return -1;
  // in place: where the input's rows lie; two results never share memory
  for (int i = 0; i < 2; ++i)
    for (int o = 0; o < 3; ++o)
      if (in[i] && in[i] == out[o] && (o == 2 || !same_rows({{d->rows, steps[i][0], steps[o + 2][0]}, {d->heads, steps[i][1], steps[o + 2][1]}}))) return -1;
  if ((sum && sum == y) || (out[2] && (out[2] == sum || out[2] == y))) return -1;
  if (!have_device("odla_b200_rms_norm")) return -2;
  RmsNorm n{};
  n.dt = kStorage[d->dtype]; n.weight_dt = kStorage[d->weight_dtype];
  n.heads = d->heads; n.channels = d->channels; n.quant = d->quant; n.group = d->group;
  n.total = (unsigned)((long long)d->rows * d->heads);
  n.epsilon = d->epsilon; n.weight_offset = d->weight_offset;
  for (int i = 0; i < 5; ++i) { n.row[i] = steps[i][0]; n.head[i] = steps[i][1]; }
  n.x = x; n.residual = residual; n.weight = weight; n.sum = sum; n.y = y; n.quantised = quantised; n.scales = scales;
  return rms_norm(n, (cudaStream_t)stream);
}

extern "C" int odla_b200_chunk_attention(const odla_b200_paged_cache* c, const void* key_cache, const void* value_cache, const odla_b200_chunk_attention_desc* d, const void* q,
                                         const int* starts, const int* prefix_pages, const int* page_table, const int* lengths, void* y, void* stream) {
  if (!cache_ok(c) || !d || c->dtype == 0 || (c->channels != 64 && c->channels != 128)) return -1;
  if (d->batch < 0 || d->tokens < 0 || d->heads < 1 || d->heads > 1024 || d->heads % c->heads || d->prefix_length < 0 || d->table_width < 0 || !std::isfinite(d->scale)) return -1;
  if (!strides_ok({{d->tokens, d->q_token}, {d->heads, d->q_head}}) || !strides_ok({{d->tokens, d->y_token}, {d->heads, d->y_head}})) return -1;
  if (!apart(c->channels, {{d->tokens, d->y_token}, {d->heads, d->y_head}})) return -1;
  for (long long s : {c->page, c->head, c->token, d->q_token, d->q_head, d->y_token, d->y_head})
    if (s % 8) return -1;
  // positions and rows (tokens and query heads) are counted in 32 bits
  if ((long long)d->table_width * c->page_size + d->prefix_length >= (1ll << 30) || d->batch >= (1 << 20) || d->tokens >= (1 << 24) || (long long)d->tokens * d->heads >= (1ll << 28)) return -1;
  if (d->batch == 0 || d->tokens == 0) return 0;
  if (!key_cache || !value_cache || !q || !y || !starts || !lengths || (d->prefix_length && !prefix_pages) || (d->table_width && !page_table)) return -1;
  if (!aligned16({key_cache, value_cache, q, y}) || (uintptr_t)starts % 4 || (uintptr_t)prefix_pages % 4 || (uintptr_t)page_table % 4 || (uintptr_t)lengths % 4) return -1;
  if (q == y && !same_rows({{d->tokens, d->q_token, d->y_token}, {d->heads, d->q_head, d->y_head}})) return -1;
  if (!have_device("odla_b200_chunk_attention")) return -2;
  const ChunkAttention a{kStorage[c->dtype], d->batch, d->tokens, d->heads, c->heads, c->channels, c->pages, c->page_size, d->prefix_length, d->table_width, d->scale,
                         c->page, c->head, c->token, d->q_token, d->q_head, d->y_token, d->y_head, key_cache, value_cache, q, starts, prefix_pages, page_table, lengths, y};
  return chunk_attention(a, (cudaStream_t)stream);
}

extern "C" int odla_b200_log_probs(const odla_b200_log_probs_desc* d, const void* logits, const float* temperature, const int* tokens, float* token_log_probs, float* entropy,
                                   int* top_tokens, float* top_log_probs, void* stream) {
  if (!d || d->dtype < 0 || d->dtype > 2 || d->rows < 0 || d->rows > (1 << 24) || d->vocab < 1 || d->vocab > kMaxVocab || d->given < 0 || d->given > kMaxVocab || d->top < 0 ||
      d->top > kMaxTop || !strides_ok({{d->rows, d->row}}))
    return -1;
  if (d->rows == 0) return 0;
  if (!logits || !element_aligned(d->dtype, {logits}) || (d->given && (!tokens || !token_log_probs)) || (d->top && (!top_tokens || !top_log_probs))) return -1;
  for (const void* p : {(const void*)temperature, (const void*)tokens, (const void*)token_log_probs, (const void*)entropy, (const void*)top_tokens, (const void*)top_log_probs})
    if ((uintptr_t)p % 4) return -1;
  if (!have_device("odla_b200_log_probs")) return -2;
  return log_probs(LogProbs{kStorage[d->dtype], d->rows, d->vocab, d->given, d->top, d->row, logits, temperature, tokens, token_log_probs, entropy, top_tokens, top_log_probs},
                   (cudaStream_t)stream);
}
