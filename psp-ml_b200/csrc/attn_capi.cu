// attn_capi.cu - C entry points of the attention operators: argument checks,
// rotary frequencies and the choice of kernel.
#include <algorithm>
#include <cmath>
#include <new>
#include <string>
#include <vector>

#include "attention.h"
#include "runtime.h"

namespace pspml {

namespace {

constexpr int kMaxHeadDim = 256;     // attention
constexpr int kMaxRotaryDim = 1024;

int bad(const std::string& msg) { return set_error(PSPML_ERR_INVALID_ARG, msg); }

int dtype_bytes(int32_t t) {
  switch (t) {
    case PSPML_DTYPE_F32: return 4;
    case PSPML_DTYPE_F16:
    case PSPML_DTYPE_BF16: return 2;
    case PSPML_DTYPE_S8: return 1;
    default: return 0;
  }
}

// Index and log-sum-exp arrays are read and written as whole elements.
template <typename T>
int check_array(const T* p, const char* name) {
  return reinterpret_cast<uintptr_t>(p) % sizeof(T) == 0
             ? PSPML_OK
             : bad(std::string(name) + ": not aligned to its element size");
}

// A view's own consistency.  Output views also have to give every element
// an address of its own.
int check_heads(const pspml_heads* h, const char* name, int64_t tokens, bool output) {
  const std::string n(name);
  if (h == nullptr) return bad(n + ": null view");
  const int bytes = dtype_bytes(h->dtype);
  if (bytes == 0) return bad(n + ": unknown dtype");
  if (h->heads <= 0 || h->head_dim <= 0) return bad(n + ": non-positive heads or head_dim");
  if (h->token_stride < 0 || h->head_stride < 0) return bad(n + ": negative stride");
  if (h->reserved != 0) return bad(n + ": reserved field is not 0");
  if (h->data == nullptr && tokens > 0) return bad(n + ": null data");
  if (reinterpret_cast<uintptr_t>(h->data) % bytes != 0)
    return bad(n + ": data is not aligned to its element size");
  if (h->dtype == PSPML_DTYPE_S8 &&
      (!(h->scale > 0.0f) || !std::isfinite(h->scale) || h->zero_point < -128 ||
       h->zero_point > 127))
    return bad(n + ": S8 needs a positive finite scale and a zero point within int8");
  if (output && tokens > 0) {
    // Spans of the inner dimension must fit in the stride of the outer one.
    const bool heads_inner = h->heads == 1 || h->head_stride >= h->head_dim;
    const bool tokens_inner = tokens == 1 || h->token_stride >= h->head_dim;
    const bool by_token =
        heads_inner && (tokens == 1 ||
                        h->token_stride >= (h->heads - 1) * h->head_stride + h->head_dim);
    const bool by_head =
        tokens_inner && (h->heads == 1 ||
                         h->head_stride >= (tokens - 1) * h->token_stride + h->head_dim);
    if (!by_token && !by_head) return bad(n + ": output elements overlap");
  }
  return PSPML_OK;
}

int check_cache(const pspml_kv_cache* c, bool written) {
  if (c == nullptr) return bad("null cache");
  if (c->dtype != PSPML_DTYPE_F32 && c->dtype != PSPML_DTYPE_F16 && c->dtype != PSPML_DTYPE_BF16)
    return bad("cache: dtype is not F32, F16 or BF16");
  const int bytes = dtype_bytes(c->dtype);
  if (c->heads <= 0 || c->head_dim <= 0 || c->page_size <= 0 || c->pages < 0)
    return bad("cache: non-positive heads, head_dim or page_size, or negative pages");
  if (c->page_stride < 0 || c->slot_stride < 0 || c->head_stride < 0)
    return bad("cache: negative stride");
  if (c->pages > 0 && (c->k == nullptr || c->v == nullptr)) return bad("cache: null pool");
  if (reinterpret_cast<uintptr_t>(c->k) % bytes != 0 || reinterpret_cast<uintptr_t>(c->v) % bytes != 0)
    return bad("cache: a pool is not aligned to its element size");
  if (c->pages > INT32_MAX) return bad("cache: more than 2^31 - 1 pages");
  if (written) {
    const int64_t dim = c->head_dim, heads = c->heads, slots = c->page_size;
    const bool by_slot = (heads == 1 || c->head_stride >= dim) &&
                         (slots == 1 || c->slot_stride >= (heads - 1) * c->head_stride + dim);
    const bool by_head = (slots == 1 || c->slot_stride >= dim) &&
                         (heads == 1 || c->head_stride >= (slots - 1) * c->slot_stride + dim);
    const int64_t span = (slots - 1) * c->slot_stride + (heads - 1) * c->head_stride + dim;
    if ((!by_slot && !by_head) || (c->pages > 1 && c->page_stride < span))
      return bad("cache: elements overlap");
  }
  return PSPML_OK;
}

int check_rotary_desc(const pspml_rotary_desc* d) {
  if (d == nullptr) return bad("null rotary descriptor");
  if (d->head_dim < 1 || d->head_dim > kMaxRotaryDim)
    return bad("rotary: head_dim must be 1 .. 1024");
  if (d->rot_dim < 0 || d->rot_dim > d->head_dim || d->rot_dim % 2 != 0)
    return bad("rotary: rot_dim must be even and at most head_dim");
  if (d->layout != PSPML_ROTARY_HALF && d->layout != PSPML_ROTARY_INTERLEAVED)
    return bad("rotary: unknown layout");
  if (!(d->base > 0.0) || !std::isfinite(d->base)) return bad("rotary: base must be positive");
  if (!std::isfinite(static_cast<float>(d->amplitude)))  // the kernels' type
    return bad("rotary: amplitude must be finite");
  if (d->scaling < PSPML_ROTARY_SCALE_NONE || d->scaling > PSPML_ROTARY_SCALE_PARTS)
    return bad("rotary: unknown scaling");
  if (d->scaling != PSPML_ROTARY_SCALE_NONE && (!(d->factor > 0.0) || !std::isfinite(d->factor)))
    return bad("rotary: factor must be positive");
  if (d->scaling == PSPML_ROTARY_SCALE_BASE && d->rot_dim == 2)
    return bad("rotary: base scaling needs rot_dim above 2");
  if (d->scaling == PSPML_ROTARY_SCALE_PARTS &&
      (!(d->original_len > 0.0) || !std::isfinite(d->original_len) || !(d->high > d->low) ||
       !std::isfinite(d->high) || !std::isfinite(d->low)))
    return bad("rotary: scaling by parts needs original_len > 0 and high > low");
  return PSPML_OK;
}

// False if a frequency is not finite: a base or factor too small for doubles.
bool frequencies(const pspml_rotary_desc& d, unsigned long long* out) {
  const double two_pi = 6.283185307179586476925286766559;
  double base = d.base;
  if (d.scaling == PSPML_ROTARY_SCALE_BASE)
    base *= std::pow(d.factor, d.rot_dim / (d.rot_dim - 2.0));
  for (int i = 0; i < d.rot_dim / 2; ++i) {
    double f = std::pow(base, -2.0 * i / d.rot_dim);
    if (d.scaling == PSPML_ROTARY_SCALE_LINEAR) f /= d.factor;
    if (d.scaling == PSPML_ROTARY_SCALE_PARTS) {
      const double r = d.original_len * f / two_pi;
      const double keep = std::fmin(1.0, std::fmax(0.0, (r - d.low) / (d.high - d.low)));
      f = keep * f + (1.0 - keep) * f / d.factor;
    }
    if (!std::isfinite(f)) return false;
    double turns = f / two_pi;
    turns -= std::floor(turns);
    // turns < 1 has 53 bits: the product with 2^64 is exact but may round up
    // to a whole turn only if turns did, which floor excludes.
    out[i] = static_cast<unsigned long long>(std::ldexp(turns, 64));
  }
  return true;
}

RotaryView view_of(const pspml_heads* in, const pspml_heads* out) {
  RotaryView v{};
  if (in == nullptr) return v;
  v.in = in->data;
  v.in_token = in->token_stride;
  v.in_head = in->head_stride;
  v.heads = in->heads;
  if (out != nullptr) {
    v.out = out->data;
    v.out_token = out->token_stride;
    v.out_head = out->head_stride;
  }
  return v;
}

int check_rotary_pair(const pspml_rotary* r, const pspml_heads* in, const pspml_heads* out,
                      int64_t tokens, const char* name) {
  const std::string n(name);
  int st = check_heads(in, name, tokens, false);
  if (st) return st;
  if (in->head_dim != r->d.head_dim) return bad(n + ": head_dim differs from the rotary's");
  if (out == nullptr) return PSPML_OK;
  st = check_heads(out, (n + " output").c_str(), tokens, true);
  if (st) return st;
  if (out->dtype == PSPML_DTYPE_S8) return bad(n + " output: S8 is not an output type here");
  if (out->heads != in->heads || out->head_dim != in->head_dim)
    return bad(n + ": input and output shapes differ");
  if (out->data == in->data && tokens > 0 &&
      (out->dtype != in->dtype || out->token_stride != in->token_stride ||
       out->head_stride != in->head_stride))
    return bad(n + ": in-place output must be the input's own view");
  return PSPML_OK;
}

// Types agree over the views that share a kernel.
int same_quant(const pspml_heads* a, const pspml_heads* b, const char* what) {
  if (a->dtype != b->dtype ||
      (a->dtype == PSPML_DTYPE_S8 && (a->scale != b->scale || a->zero_point != b->zero_point)))
    return bad(std::string(what) + ": types or quantisation differ");
  return PSPML_OK;
}

void fill_rotary(const pspml_rotary* r, int64_t tokens, const int32_t* positions,
                 const pspml_heads* any_in, int32_t out_dtype, RotaryArgs* a) {
  a->positions = positions;
  a->freq = r->freq;
  a->tokens = tokens;
  a->dim = r->d.head_dim;
  a->rot = r->d.rot_dim;
  a->layout = r->d.layout;
  a->amplitude = static_cast<float>(r->d.amplitude);
  a->in_dtype = any_in->dtype;
  a->out_dtype = out_dtype;
  a->scale = any_in->dtype == PSPML_DTYPE_S8 ? any_in->scale : 1.0f;
  a->zero = any_in->dtype == PSPML_DTYPE_S8 ? any_in->zero_point : 0;
}

int check_attention(const pspml_ctx* ctx, const pspml_attention_desc* d, int64_t tokens,
                    int32_t sequences, const int32_t* starts, const pspml_heads* q,
                    const pspml_heads* out, const float* lse) {
  if (ctx == nullptr) return bad("null context");
  if (d == nullptr) return bad("null attention descriptor");
  if (!std::isfinite(d->scale)) return bad("attention: scale must be finite");
  if (d->causal != 0 && d->causal != 1) return bad("attention: causal must be 0 or 1");
  if (d->window < 0 || (d->window > 0 && !d->causal))
    return bad("attention: window must be 0, or positive and causal");
  if (d->reserved != 0) return bad("attention: reserved field is not 0");
  if (tokens < 0 || tokens > INT32_MAX) return bad("attention: tokens must be 0 .. 2^31 - 1");
  if (sequences < 0) return bad("attention: negative number of sequences");
  if (starts == nullptr && sequences > 0) return bad("attention: null starts");
  int st = check_array(starts, "starts");
  if (st) return st;
  if ((st = check_array(lse, "lse"))) return st;
  if ((st = check_heads(q, "q", tokens, false))) return st;
  if ((st = check_heads(out, "out", tokens, true))) return st;
  if (q->dtype == PSPML_DTYPE_S8) return bad("q: S8 is not an attention input type");
  if (q->head_dim > kMaxHeadDim)
    return set_error(PSPML_ERR_UNSUPPORTED, "attention: head_dim above 256");
  if (out->heads != q->heads || out->head_dim != q->head_dim)
    return bad("attention: q and out shapes differ");
  if (out->dtype != q->dtype && out->dtype != PSPML_DTYPE_S8)
    return bad("attention: out must have q's dtype or S8");
  if (tokens * q->heads > INT32_MAX)
    return set_error(PSPML_ERR_UNSUPPORTED, "attention: more than 2^31 - 1 rows");
  return PSPML_OK;
}

void fill_attention(const pspml_attention_desc* d, int64_t tokens, int32_t sequences,
                    const int32_t* starts, const pspml_heads* q, const pspml_heads* out,
                    float* lse, AttnArgs* a) {
  a->q = q->data;
  a->out = out->data;
  a->lse = lse;
  a->starts = starts;
  a->tokens = tokens;
  a->sequences = sequences;
  a->q_token = q->token_stride;
  a->q_head = q->head_stride;
  a->o_token = out->token_stride;
  a->o_head = out->head_stride;
  a->q_heads = q->heads;
  a->dim = q->head_dim;
  a->causal = d->causal;
  a->window = d->window;
  a->scale = d->scale;
  a->dtype = q->dtype;
  a->out_dtype = out->dtype;
  a->out_inv_scale = out->dtype == PSPML_DTYPE_S8 ? 1.0f / out->scale : 1.0f;
  a->out_zero = out->dtype == PSPML_DTYPE_S8 ? out->zero_point : 0;
}

bool aligned(const void* p, int64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0;
}

// What the tensor-core kernels' 16-byte loads and 8-element stores need.
bool vector_form(const AttnArgs& a) {
  if (a.dtype == PSPML_DTYPE_F32 || a.dim > 128 || a.dim % 8 != 0) return false;
  const int out_bytes = a.out_dtype == PSPML_DTYPE_S8 ? 8 : 16;
  return aligned(a.q, 16) && aligned(a.k, 16) && aligned(a.v, 16) && aligned(a.out, out_bytes) &&
         (a.q_token | a.q_head | a.kv_token | a.kv_head | a.v_token | a.v_head | a.page_stride |
          a.o_token | a.o_head) % 8 == 0;
}

// Split calls of one context run one after another whatever streams they are
// given, since they share its workspace.  Every call waits for the last one's
// event, also on an equal handle, which need not be the same stream: each host
// thread has a default stream of its own under one handle, and a destroyed
// stream's handle may come back while its work runs.  Under capture an event of
// the outside cannot be waited for: there the caller keeps the order.
int with_workspace(pspml_ctx* ctx, const AttnArgs& a, cudaStream_t s,
                   cudaError_t (*launch)(const AttnArgs&, const AttnWork&, cudaStream_t)) {
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  int st = cuda_status(cudaStreamIsCapturing(s, &capture), "cudaStreamIsCapturing");
  if (st) return st;
  const bool order = capture == cudaStreamCaptureStatusNone;
  if (ctx->attn_workspace == nullptr) {
    if (!order)
      return set_error(PSPML_ERR_UNSUPPORTED,
                       "attention: a context's first call allocates and cannot be captured");
    if ((st = cuda_status(cudaMalloc(&ctx->attn_workspace, attn_workspace_bytes(ctx->num_sms)),
                          "cudaMalloc(attention workspace)")))
      return st;
  }
  AttnWork w;
  w.base = ctx->attn_workspace;
  w.counters = ctx->dev_err + 64;
  w.err = ctx->dev_err;
  w.num_sms = ctx->num_sms;
  if (order && ctx->attn_used &&
      (st = cuda_status(cudaStreamWaitEvent(s, ctx->attn_done, 0), "cudaStreamWaitEvent")))
    return st;
  if ((st = cuda_status(launch(a, w, s), "attention launch"))) return st;
  if (order) {
    if ((st = cuda_status(cudaEventRecord(ctx->attn_done, s), "cudaEventRecord"))) return st;
    ctx->attn_used = true;
  }
  return PSPML_OK;
}

// Few rows a key head: the cache's bytes bound the call (attn_step.cu); more
// rows: attn_tc.cu; what neither fits: attn_any.cu.
int run_attention(pspml_ctx* ctx, const AttnArgs& a, cudaStream_t s) {
  if (!vector_form(a)) return cuda_status(launch_attn_any(a, s), "attention launch");
  const int64_t group = a.q_heads / a.kv_heads;
  if (a.paged && a.max_new * group <= 16) return with_workspace(ctx, a, s, launch_attn_step);
  if (attn_tc_covers(a)) return with_workspace(ctx, a, s, launch_attn_tc);
  return cuda_status(launch_attn_any(a, s), "attention launch");
}

}  // namespace

}  // namespace pspml

using namespace pspml;

extern "C" {

int pspml_rotary_frequencies(const pspml_rotary_desc* d, uint64_t* host_out) {
  clear_error();
  int st = check_rotary_desc(d);
  if (st) return st;
  if (host_out == nullptr && d->rot_dim > 0) return bad("null output");
  unsigned long long f[kMaxRotaryDim / 2];
  if (!frequencies(*d, f)) return bad("rotary: a frequency is not finite");
  std::copy_n(f, d->rot_dim / 2, host_out);
  return PSPML_OK;
}

int pspml_rotary_create(pspml_ctx* ctx, const pspml_rotary_desc* d, pspml_rotary** out) {
  clear_error();
  if (out == nullptr) return bad("null output pointer");
  *out = nullptr;
  if (ctx == nullptr) return bad("null context");
  int st = check_rotary_desc(d);
  if (st) return st;
  unsigned long long f[kMaxRotaryDim / 2];
  if (!frequencies(*d, f)) return bad("rotary: a frequency is not finite");
  if ((st = cuda_status(cudaSetDevice(ctx->device), "cudaSetDevice"))) return st;
  auto* r = new (std::nothrow) pspml_rotary();
  if (r == nullptr) return set_error(PSPML_ERR_OOM, "host allocation failed");
  r->device = ctx->device;
  r->num_sms = ctx->num_sms;
  r->d = *d;
  const size_t bytes = d->rot_dim / 2 * sizeof(f[0]);
  if (bytes > 0) {
    st = cuda_status(cudaMalloc(&r->freq, bytes), "cudaMalloc(rotary)");
    // Uploaded on the context's stream and waited for: calls on any stream
    // may follow.
    if (!st)
      st = cuda_status(cudaMemcpyAsync(r->freq, f, bytes, cudaMemcpyHostToDevice, ctx->stream),
                       "rotary upload");
    if (!st) st = cuda_status(cudaStreamSynchronize(ctx->stream), "rotary upload");
  }
  if (st) {
    if (r->freq) cudaFree(r->freq);
    delete r;
    return st;
  }
  *out = r;
  return PSPML_OK;
}

int pspml_rotary_destroy(pspml_rotary* r) {
  if (r == nullptr) return PSPML_OK;
  cudaSetDevice(r->device);
  if (r->freq) cudaFree(r->freq);
  delete r;
  return PSPML_OK;
}

int pspml_rotary_apply(pspml_rotary* r, int64_t tokens, const int32_t* positions,
                       const pspml_heads* q, const pspml_heads* q_out, const pspml_heads* k,
                       const pspml_heads* k_out, void* stream) {
  clear_error();
  if (r == nullptr) return bad("null rotary");
  if (tokens < 0) return bad("negative number of tokens");
  if (positions == nullptr && tokens > 0) return bad("null positions");
  if ((k == nullptr) != (k_out == nullptr)) return bad("k and k_out go together");
  if (q_out == nullptr) return bad("null q output");
  int st = check_array(positions, "positions");
  if (st) return st;
  if ((st = check_rotary_pair(r, q, q_out, tokens, "q"))) return st;
  if (k != nullptr) {
    if ((st = check_rotary_pair(r, k, k_out, tokens, "k")) || (st = same_quant(q, k, "q and k")))
      return st;
    if (q_out->dtype != k_out->dtype) return bad("q and k outputs: types differ");
  }
  if (tokens == 0) return PSPML_OK;
  RotaryArgs a{};
  a.q = view_of(q, q_out);
  a.k = view_of(k, k_out);
  fill_rotary(r, tokens, positions, q, q_out->dtype, &a);
  if ((st = cuda_status(cudaSetDevice(r->device), "cudaSetDevice"))) return st;
  return cuda_status(launch_rotary(a, r->num_sms, static_cast<cudaStream_t>(stream)),
                     "rotary launch");
}

int pspml_rotary_append(pspml_rotary* r, int64_t tokens, const int32_t* positions,
                        const int64_t* slots, const pspml_heads* q, const pspml_heads* q_out,
                        const pspml_heads* k, const pspml_heads* v, const pspml_kv_cache* cache,
                        void* stream) {
  clear_error();
  if (r == nullptr) return bad("null rotary");
  if (tokens < 0) return bad("negative number of tokens");
  if ((positions == nullptr || slots == nullptr) && tokens > 0)
    return bad("null positions or slots");
  if ((q == nullptr) != (q_out == nullptr)) return bad("q and q_out go together");
  int st = check_array(positions, "positions");
  if (st) return st;
  if ((st = check_array(slots, "slots"))) return st;
  if ((st = check_cache(cache, true))) return st;
  if ((st = check_rotary_pair(r, k, nullptr, tokens, "k"))) return st;
  if ((st = check_rotary_pair(r, v, nullptr, tokens, "v"))) return st;
  if ((st = same_quant(k, v, "k and v"))) return st;
  if (k->heads != cache->heads || v->heads != cache->heads || cache->head_dim != k->head_dim)
    return bad("k, v and the cache: shapes differ");
  if (q != nullptr) {
    if ((st = check_rotary_pair(r, q, q_out, tokens, "q")) || (st = same_quant(q, k, "q and k")))
      return st;
    if (q_out->dtype != cache->dtype) return bad("q output and cache: types differ");
  }
  if (tokens == 0) return PSPML_OK;
  RotaryArgs a{};
  a.q = view_of(q, q_out);
  a.k = view_of(k, nullptr);
  a.v = view_of(v, nullptr);
  a.k.out = cache->k;
  a.v.out = cache->v;
  a.k.out_head = a.v.out_head = cache->head_stride;
  a.slots = slots;
  a.page_stride = cache->page_stride;
  a.slot_stride = cache->slot_stride;
  a.page_size = cache->page_size;
  a.slots_total = cache->pages * cache->page_size;
  fill_rotary(r, tokens, positions, k, cache->dtype, &a);
  if ((st = cuda_status(cudaSetDevice(r->device), "cudaSetDevice"))) return st;
  return cuda_status(launch_rotary(a, r->num_sms, static_cast<cudaStream_t>(stream)),
                     "rotary launch");
}

int pspml_attention_prompt(pspml_ctx* ctx, const pspml_attention_desc* d, int64_t tokens,
                           int32_t sequences, const int32_t* starts, const pspml_heads* q,
                           const pspml_heads* k, const pspml_heads* v, const pspml_heads* out,
                           float* lse, void* stream) {
  clear_error();
  int st = check_attention(ctx, d, tokens, sequences, starts, q, out, lse);
  if (st) return st;
  if ((st = check_heads(k, "k", tokens, false)) || (st = check_heads(v, "v", tokens, false)))
    return st;
  if (k->dtype != q->dtype || v->dtype != q->dtype) return bad("q, k and v: types differ");
  if (k->heads != v->heads || k->head_dim != q->head_dim || v->head_dim != q->head_dim ||
      q->heads % k->heads != 0)
    return bad("q, k and v: shapes do not go together");
  if (tokens == 0 || sequences == 0) return PSPML_OK;
  AttnArgs a{};
  fill_attention(d, tokens, sequences, starts, q, out, lse, &a);
  a.k = k->data;
  a.v = v->data;
  a.kv_heads = k->heads;
  a.kv_token = k->token_stride;
  a.kv_head = k->head_stride;
  a.v_token = v->token_stride;
  a.v_head = v->head_stride;
  if ((st = cuda_status(cudaSetDevice(ctx->device), "cudaSetDevice"))) return st;
  return run_attention(ctx, a, static_cast<cudaStream_t>(stream));
}

int pspml_attention_cached(pspml_ctx* ctx, const pspml_attention_desc* d, int64_t tokens,
                           int32_t sequences, int32_t max_new, const int32_t* starts,
                           const int32_t* lengths, const int32_t* pages, int64_t pages_stride,
                           const pspml_heads* q, const pspml_kv_cache* cache,
                           const pspml_heads* out, float* lse, void* stream) {
  clear_error();
  int st = check_attention(ctx, d, tokens, sequences, starts, q, out, lse);
  if (st) return st;
  if ((st = check_cache(cache, false))) return st;
  if (max_new < 0) return bad("negative max_new");
  if (pages_stride < 0) return bad("negative pages_stride");
  if (sequences > 0 && (lengths == nullptr || (pages == nullptr && pages_stride > 0)))
    return bad("null lengths or pages");
  if ((st = check_array(lengths, "lengths")) || (st = check_array(pages, "pages"))) return st;
  if (cache->dtype != q->dtype) return bad("q and the cache: types differ");
  if (cache->head_dim != q->head_dim || q->heads % cache->heads != 0)
    return bad("q and the cache: shapes do not go together");
  if (tokens == 0 || sequences == 0 || max_new == 0) return PSPML_OK;
  AttnArgs a{};
  fill_attention(d, tokens, sequences, starts, q, out, lse, &a);
  a.k = cache->k;
  a.v = cache->v;
  a.kv_heads = cache->heads;
  a.kv_token = a.v_token = cache->slot_stride;
  a.kv_head = a.v_head = cache->head_stride;
  a.page_stride = cache->page_stride;
  a.page_size = cache->page_size;
  a.n_pages = cache->pages;
  a.lengths = lengths;
  a.pages = pages;
  a.pages_stride = pages_stride;
  a.max_new = max_new;
  a.paged = 1;
  if ((st = cuda_status(cudaSetDevice(ctx->device), "cudaSetDevice"))) return st;
  return run_attention(ctx, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
