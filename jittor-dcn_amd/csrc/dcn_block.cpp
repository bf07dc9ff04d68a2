// dcn_block.cpp — entry points of the residual block's operators (include/dcn.h): argument
// checks, then one launcher each. Nothing here allocates, synchronises or keeps state, so every
// call can be captured into a graph.
#include <algorithm>
#include <cmath>
#include <string>

#include "dcn_block.h"
#include "dcn_philox.h"

extern "C" __attribute__((visibility("hidden"))) int dcn_internal_fail(int code, const char* msg);
extern "C" __attribute__((visibility("hidden"))) int dcn_internal_bind(dcn_handle* h,
                                                                      void** stream);

namespace {

int fail(int code, const char* msg) { return dcn_internal_fail(code, msg); }

int done(hipError_t e, const char* what) {
  if (e == hipSuccess) return DCN_OK;
  return fail(DCN_ERR_HIP, (std::string(what) + ": " + hipGetErrorString(e)).c_str());
}

// The handle's device for one call, the caller's current device afterwards.
struct DeviceScope {
  int prev = -1;
  hipStream_t stream = nullptr;
  int bind(dcn_handle* h) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    void* s = nullptr;
    const int rc = dcn_internal_bind(h, &s);
    stream = static_cast<hipStream_t>(s);
    return rc;
  }
  ~DeviceScope() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
};

bool dtype_ok(int dt) { return dt == DCN_F32 || dt == DCN_BF16; }
size_t dtype_bytes(int dt) { return dt == DCN_BF16 ? 2 : 4; }
bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// [a, a + na) and [b, b + nb) share a byte (null pointers never do)
bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  if (!a || !b || !na || !nb) return false;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + nb && y < x + na;
}

// Threshold and scale of a drop probability (include/dcn.h).
bool drop_args(float p, uint64_t seed, uint64_t offset, const void* rng, dcn::DropArgs* a) {
  if (!(p >= 0.f && p <= 1.f)) return false;  // NaN too
  a->rng = static_cast<const uint64_t*>(rng);
  a->seed = seed;
  a->offset = offset;
  a->thr = (unsigned)std::floor((double)p * 65536.0 + 0.5);
  a->scale = a->thr < 65536u ? (float)(65536.0 / (double)(65536u - a->thr)) : 0.f;
  return true;
}

int dropout(dcn_handle* h, const dcn_dropout_desc* d, const void* x, const void* res, void* y,
            const void* rng) {
  if (!d) return fail(DCN_ERR_INVALID, "null descriptor");
  if (!dtype_ok(d->dtype)) return fail(DCN_ERR_INVALID, "unknown dtype");
  if (d->n < 0 || d->n > (1LL << 46)) return fail(DCN_ERR_INVALID, "bad element count");
  if (d->group < 1) return fail(DCN_ERR_INVALID, "group must be positive");
  dcn::DropArgs a;
  if (!drop_args(d->p, d->seed, d->offset, rng, &a))
    return fail(DCN_ERR_INVALID, "dropout needs 0 <= p <= 1");
  if (!aligned(rng, 8)) return fail(DCN_ERR_INVALID, "rng must be 8-byte aligned");
  const size_t es = dtype_bytes(d->dtype), bytes = (size_t)d->n * es;
  if (d->n > 0 && (!x || !y)) return fail(DCN_ERR_INVALID, "null tensor");
  for (const void* p : {x, res, static_cast<const void*>(y)})
    if (!aligned(p, es)) return fail(DCN_ERR_INVALID, "tensor not aligned to its elements");
  if ((y != x && overlap(y, bytes, x, bytes)) || (y != res && overlap(y, bytes, res, bytes)) ||
      overlap(y, bytes, rng, 16))
    return fail(DCN_ERR_INVALID, "the output overlaps an input");
  DeviceScope ds;
  if (int rc = ds.bind(h)) return rc;
  return done(dcn::launch_dropout(a, d->dtype, x, res, y, (uint64_t)d->n, (uint64_t)d->group,
                                  ds.stream),
              "dropout");
}

// The checks that need no tensor; fills the geometry of `a`.
int block_geo(const dcn_block_desc* d, dcn::BlockArgs* a) {
  if (!d) return fail(DCN_ERR_INVALID, "null descriptor");
  *a = dcn::BlockArgs{};
  if (d->B <= 0 || d->C <= 0 || d->P <= 0) return fail(DCN_ERR_INVALID, "B, C, P must be positive");
  if (!dtype_ok(d->dtype)) return fail(DCN_ERR_INVALID, "unknown dtype");
  if (d->layout != DCN_NCHW && d->layout != DCN_NHWC) return fail(DCN_ERR_INVALID, "unknown layout");
  if ((double)d->B * d->C * d->P > (double)(1LL << 40) || (long long)d->B * d->P > (1LL << 34) ||
      d->C > (1 << 23) || d->P > (1 << 30))
    return fail(DCN_ERR_UNSUPPORTED,
                "more than 2^40 elements or 2^34 positions, C above 2^23 or P above 2^30");
  for (int k : {d->post, d->pre})
    if (k < DCN_NORM_NONE || k > DCN_NORM_LAYER) return fail(DCN_ERR_INVALID, "unknown norm");
  if (d->gate < DCN_GATE_NONE || d->gate > DCN_GATE_IMAGE)
    return fail(DCN_ERR_INVALID, "unknown gate kind");
  if (d->gate_act < DCN_ACT_LINEAR || d->gate_act > DCN_ACT_SILU)
    return fail(DCN_ERR_INVALID, "unknown gate activation");
  for (float e : {d->eps_post, d->eps_pre})
    if (!(e >= 0.f && std::isfinite(e))) return fail(DCN_ERR_INVALID, "eps must be finite and >= 0");
  if (d->drop_image != 0 && d->drop_image != 1) return fail(DCN_ERR_INVALID, "drop_image is 0 or 1");
  a->B = d->B; a->C = d->C; a->P = d->P;
  a->layout = d->layout; a->dtype = d->dtype;
  a->post = d->post; a->pre = d->pre;
  a->gate_kind = d->gate; a->act = d->gate_act;
  a->drop_image = d->drop_image;
  a->eps1 = d->eps_post; a->eps2 = d->eps_pre; a->alpha = d->alpha;
  return DCN_OK;
}

// The inputs of either direction.
int block_inputs(const dcn_block_desc* d, const dcn_block_io* io, dcn::BlockArgs* a) {
  if (int rc = block_geo(d, a)) return rc;
  if (!io) return fail(DCN_ERR_INVALID, "null tensor list");
  if (!drop_args(d->drop_p, d->seed, d->offset, io->rng, &a->drop))
    return fail(DCN_ERR_INVALID, "dropout needs 0 <= p <= 1");
  if (!aligned(io->rng, 8)) return fail(DCN_ERR_INVALID, "rng must be 8-byte aligned");
  if (!io->x && !io->residual) return fail(DCN_ERR_INVALID, "neither x nor a residual");
  if (!io->x && (d->post || d->gate || io->scale || io->w_post || io->b_post || d->drop_p > 0.f))
    return fail(DCN_ERR_INVALID, "post norm, gate, scale and dropout need x");
  if (!io->x && !d->pre) return fail(DCN_ERR_INVALID, "nothing to compute: no x and no pre norm");
  if ((io->w_post || io->b_post) && !d->post) return fail(DCN_ERR_INVALID, "w_post / b_post without a post norm");
  if ((io->w_pre || io->b_pre) && !d->pre) return fail(DCN_ERR_INVALID, "w_pre / b_pre without a pre norm");
  if ((io->gate != nullptr) != (d->gate != DCN_GATE_NONE))
    return fail(DCN_ERR_INVALID, "the gate tensor and the gate kind must come together");
  a->x = io->x; a->res = io->residual; a->gate = io->gate; a->scale = io->scale;
  if (!aligned(io->stats, 16)) return fail(DCN_ERR_INVALID, "stats must be 16-byte aligned");
  a->stats = io->stats;
  a->w1 = io->w_post; a->b1 = io->b_post; a->w2 = io->w_pre; a->b2 = io->b_pre;
  return DCN_OK;
}

struct Span {
  const void* p;
  size_t bytes;
};

// Every output apart from every input and every other output; `inplace_out` may be `inplace_in`,
// byte for byte.
int block_spans(const Span* in, int nin, const Span* out, int nout, size_t es,
                const void* inplace_out, const void* inplace_in) {
  for (int i = 0; i < nin; ++i)
    if (!aligned(in[i].p, es)) return fail(DCN_ERR_INVALID, "tensor not aligned to its elements");
  for (int i = 0; i < nout; ++i) {
    if (!aligned(out[i].p, es)) return fail(DCN_ERR_INVALID, "tensor not aligned to its elements");
    for (int j = 0; j < nin; ++j) {
      if (out[i].p && out[i].p == inplace_out && in[j].p == inplace_in && out[i].p == in[j].p &&
          out[i].bytes == in[j].bytes)
        continue;
      if (overlap(out[i].p, out[i].bytes, in[j].p, in[j].bytes))
        return fail(DCN_ERR_INVALID, "an output overlaps an input");
    }
    for (int j = 0; j < i; ++j)
      if (overlap(out[i].p, out[i].bytes, out[j].p, out[j].bytes))
        return fail(DCN_ERR_INVALID, "two outputs overlap");
  }
  return DCN_OK;
}

size_t up128(size_t v) { return (v + 127) / 128 * 128; }

// Bytes of an 8-bit matrix of `rows` x K (K a multiple of 128) and of its exponents.
size_t fp8_bytes(size_t rows, size_t k) { return rows * k; }
size_t exp_bytes(size_t rows, size_t k, int block) {
  return k / 128 * (block == 128 ? (rows + 127) / 128 : up128(rows));
}

int fp8_pair(const void* q, const void* s, const char* what) {
  if ((q != nullptr) != (s != nullptr))
    return fail(DCN_ERR_INVALID, (std::string(what) + ": bytes and exponents come together").c_str());
  if (!aligned(q, 16) || !aligned(s, 4))
    return fail(DCN_ERR_INVALID,
                (std::string(what) + ": bytes 16-byte, exponents 4-byte aligned").c_str());
  return DCN_OK;
}

// Below 2^24 tiles of 128 x 128, one workgroup of 256 threads each: a launch takes less than 2^32
// threads. kMaxSide: the same for 512 threads per 16 rows of a product's long side.
constexpr int kMaxSide = 1 << 26;
bool tiles_ok(double a, double b, double images) {
  return std::ceil(a / 128) * std::ceil(b / 128) * images < 16777216.0;
}

int fp8_matmul_check(const dcn_fp8_matmul_desc* d) {
  if (!d) return fail(DCN_ERR_INVALID, "null descriptor");
  if (d->M <= 0 || d->N <= 0 || d->K <= 0) return fail(DCN_ERR_INVALID, "M, N, K must be positive");
  if (d->K % 128) return fail(DCN_ERR_INVALID, "K must be a multiple of 128");
  for (int b : {d->a_block, d->b_block})
    if (b != 1 && b != 128) return fail(DCN_ERR_INVALID, "exponents are per 1 or 128 rows");
  if (d->layout != DCN_NCHW && d->layout != DCN_NHWC) return fail(DCN_ERR_INVALID, "unknown layout");
  if (d->layout == DCN_NCHW && (d->P <= 0 || d->N % d->P))
    return fail(DCN_ERR_INVALID, "DCN_NCHW needs N a multiple of P");
  if (!dtype_ok(d->out_dtype)) return fail(DCN_ERR_INVALID, "unknown dtype");
  if (d->M > kMaxSide || d->N > kMaxSide || d->K > (1 << 30) || !tiles_ok(d->M, d->N, 1))
    return fail(DCN_ERR_UNSUPPORTED,
                "M or N above 2^26, K above 2^30, or 2^24 tiles of 128 x 128 of the product");
  return DCN_OK;
}

// One pointwise product: where its 8-bit operands lie in the workspaces and in `saved`.
struct Pointwise {
  size_t T, cp, op, kt;                       // tokens; C, O and the tokens by channel, up to 128s
  size_t wq, ws, xq, xs, mm, fwd;             // forward workspace
  size_t wt, wts, xc, xcs, saved;             // saved
  size_t gq, gs, gc, gcs, mmb, bwd;           // backward workspace
  bool few;
  dcn_fp8_matmul_desc y, gx, gw;
};

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

int pointwise(const dcn_fp8_pointwise_desc* d, int grads, Pointwise* p) {
  if (!d) return fail(DCN_ERR_INVALID, "null descriptor");
  if (d->B <= 0 || d->C <= 0 || d->P <= 0 || d->O <= 0)
    return fail(DCN_ERR_INVALID, "B, C, P, O must be positive");
  if (!dtype_ok(d->dtype)) return fail(DCN_ERR_INVALID, "unknown dtype");
  if (d->layout != DCN_NCHW && d->layout != DCN_NHWC) return fail(DCN_ERR_INVALID, "unknown layout");
  if (grads != DCN_FP8_SERVED && (grads & ~(DCN_FP8_GRAD_X | DCN_FP8_GRAD_W)))
    return fail(DCN_ERR_INVALID, "unknown gradient");
  const bool maps = d->layout == DCN_NCHW;
  p->T = (size_t)d->B * d->P;
  p->cp = up128(d->C);
  p->op = up128(d->O);
  p->kt = maps ? d->B * up128(d->P) : up128(p->T);
  const double widest = std::max(d->C, d->O);
  if (p->T > kMaxSide || p->kt > (1u << 30) || widest > kMaxSide ||
      // (twice: the weight's tiles and x's go in one launch)
      !tiles_ok(maps ? widest : (double)p->T, maps ? d->P : widest, maps ? 2.0 * d->B : 2) ||
      !tiles_ok(d->O, d->C, 2) || !tiles_ok((double)p->T, widest, 1))
    return fail(DCN_ERR_UNSUPPORTED, "tensor too large");
  const int T = (int)p->T;
  if (maps) {
    p->y = {d->O, T, (int)p->cp, 128, 1, DCN_NCHW, d->P, d->dtype};
    p->gx = {d->C, T, (int)p->op, 128, 1, DCN_NCHW, d->P, d->dtype};
  } else {
    p->y = {T, d->O, (int)p->cp, 1, 128, DCN_NHWC, 0, d->dtype};
    p->gx = {T, d->C, (int)p->op, 1, 128, DCN_NHWC, 0, d->dtype};
  }
  p->gw = {d->O, d->C, (int)p->kt, 1, 1, DCN_NHWC, 0, d->dtype};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += up256(bytes);
    return o;
  };
  p->few = !maps && dcn::fp8_few_tokens(p->T);  // rounded inside the product
  if (grads != DCN_FP8_SERVED) {
    p->wq = take(fp8_bytes(d->O, p->cp));
    p->ws = take(exp_bytes(d->O, p->cp, 128));
  }
  if (!p->few) {
    p->xq = take(fp8_bytes(p->T, p->cp));
    p->xs = take(exp_bytes(p->T, p->cp, 1));
    p->mm = take(dcn::fp8_matmul_ws_bytes(p->y));
  }
  p->fwd = at;
  at = 0;
  if (grads & DCN_FP8_GRAD_X) {
    p->wt = take(fp8_bytes(d->C, p->op));
    p->wts = take(exp_bytes(d->C, p->op, 128));
  }
  if (grads & DCN_FP8_GRAD_W) {
    p->xc = take(fp8_bytes(d->C, p->kt));
    p->xcs = take(exp_bytes(d->C, p->kt, 1));
  }
  p->saved = at;
  at = 0;
  if (grads & DCN_FP8_GRAD_X) {
    p->gq = take(fp8_bytes(p->T, p->op));
    p->gs = take(exp_bytes(p->T, p->op, 1));
  }
  if (grads & DCN_FP8_GRAD_W) {
    p->gc = take(fp8_bytes(d->O, p->kt));
    p->gcs = take(exp_bytes(d->O, p->kt, 1));
  }
  p->mmb = take(std::max(grads & DCN_FP8_GRAD_X ? dcn::fp8_matmul_ws_bytes(p->gx) : 0,
                         grads & DCN_FP8_GRAD_W ? dcn::fp8_matmul_ws_bytes(p->gw) : 0));
  p->bwd = at;
  return DCN_OK;
}

int buffer_ok(const void* p, size_t have, size_t need, const char* what) {
  if (need && (!p || have < need))
    return fail(DCN_ERR_WORKSPACE, (std::string(what) + " too small").c_str());
  if (!aligned(p, 256))
    return fail(DCN_ERR_INVALID, (std::string(what) + " must be 256-byte aligned").c_str());
  return DCN_OK;
}

}  // namespace

extern "C" {

int dcn_fp8_pointwise_workspace(const dcn_fp8_pointwise_desc* d, int grads, size_t* fwd_ws,
                                size_t* saved, size_t* bwd_ws) {
  Pointwise p{};
  if (int rc = pointwise(d, grads, &p)) return rc;
  if (!fwd_ws || !saved || !bwd_ws) return fail(DCN_ERR_INVALID, "null out pointer");
  *fwd_ws = p.fwd;
  *saved = p.saved;
  *bwd_ws = p.bwd;
  return DCN_OK;
}

int dcn_fp8_pointwise_fwd(dcn_handle* h, const dcn_fp8_pointwise_desc* d, int grads, const void* x,
                          const void* w, const void* q, const void* s, void* y, void* saved,
                          size_t saved_bytes, void* ws, size_t ws_bytes) {
  Pointwise p{};
  if (int rc = pointwise(d, grads, &p)) return rc;
  if (!x || !y || !(w || q)) return fail(DCN_ERR_INVALID, "null tensor");
  if (w && (q || s || grads == DCN_FP8_SERVED))
    return fail(DCN_ERR_INVALID, "one weight: as it is or in 8 bits");
  if (int rc = fp8_pair(q, s, "weight")) return rc;
  if (q && grads && grads != DCN_FP8_SERVED)
    return fail(DCN_ERR_INVALID, "a weight in 8 bits has no gradients");
  if (int rc = buffer_ok(ws, ws_bytes, p.fwd, "pointwise workspace")) return rc;
  if (int rc = buffer_ok(saved, saved_bytes, p.saved, "saved buffer")) return rc;
  const size_t es = dtype_bytes(d->dtype);
  const Span in[] = {{x, p.T * d->C * es}, {w, (size_t)d->O * d->C * es},
                     {q, fp8_bytes(d->O, p.cp)}, {s, exp_bytes(d->O, p.cp, 128)}};
  const Span out[] = {{y, p.T * d->O * es}, {p.saved ? saved : nullptr, p.saved},
                      {p.fwd ? ws : nullptr, p.fwd}};
  for (const void* t : {x, w, static_cast<const void*>(y)})
    if (!aligned(t, es)) return fail(DCN_ERR_INVALID, "tensor not aligned to its elements");
  if (int rc = block_spans(in, 4, out, 3, 1, nullptr, nullptr)) return rc;
  DeviceScope ds;
  if (int rc = ds.bind(h)) return rc;
  char *b = static_cast<char*>(ws), *k = static_cast<char*>(saved);
  const bool gx = grads & DCN_FP8_GRAD_X, gw = grads & DCN_FP8_GRAD_W;
  hipError_t e = hipSuccess;
  const bool maps = d->layout == DCN_NCHW, few = p.few, x8 = !few || gw;
  char *xq = few ? nullptr : b + p.xq, *xs = few ? nullptr : b + p.xs;
  char *xc = gw ? k + p.xc : nullptr, *xcs = gw ? k + p.xcs : nullptr;
  if (w) {
    char *wt = gx ? k + p.wt : nullptr, *wts = gx ? k + p.wts : nullptr;
    q = b + p.wq;
    s = b + p.ws;
    e = x8 ? dcn::launch_fp8_quantize_both(d->B, d->C, d->P, d->layout, d->dtype, x, xq, xs, xc, xcs,
                                           d->O, w, b + p.wq, b + p.ws, wt, wts, ds.stream)
           : dcn::launch_fp8_quantize_weight(d->O, d->C, d->dtype, w, b + p.wq, b + p.ws, wt, wts,
                                             ds.stream);
  } else if (x8) {
    e = dcn::launch_fp8_quantize(d->B, d->C, d->P, d->layout, d->dtype, x, xq, xs, xc, xcs, ds.stream);
  }
  if (e == hipSuccess && few) {
    e = dcn::launch_fp8_few_tokens(p.y, d->C, x, q, s, y, ds.stream);
  } else if (e == hipSuccess) {
    e = dcn::launch_fp8_matmul(p.y, maps ? q : b + p.xq, maps ? s : b + p.xs, maps ? b + p.xq : q,
                               maps ? b + p.xs : s, y, b + p.mm, ds.stream);
  }
  return done(e, "fp8_pointwise forward");
}

int dcn_fp8_pointwise_bwd(dcn_handle* h, const dcn_fp8_pointwise_desc* d, int grads,
                          const void* grad_y, const void* saved, size_t saved_bytes, void* grad_x,
                          void* grad_w, void* ws, size_t ws_bytes) {
  Pointwise p{};
  if (int rc = pointwise(d, grads, &p)) return rc;
  if (!grad_y || !(grad_x || grad_w)) return fail(DCN_ERR_INVALID, "null tensor");
  if ((grad_x && !(grads & DCN_FP8_GRAD_X)) || (grad_w && !(grads & DCN_FP8_GRAD_W)))
    return fail(DCN_ERR_INVALID, "the forward kept nothing for this gradient");
  if (int rc = buffer_ok(ws, ws_bytes, p.bwd, "pointwise workspace")) return rc;
  if (int rc = buffer_ok(saved, saved_bytes, p.saved, "saved buffer")) return rc;
  const size_t es = dtype_bytes(d->dtype);
  for (const void* t : {grad_y, static_cast<const void*>(grad_x), static_cast<const void*>(grad_w)})
    if (!aligned(t, es)) return fail(DCN_ERR_INVALID, "tensor not aligned to its elements");
  const Span in[] = {{grad_y, p.T * d->O * es}, {saved, p.saved}};
  const Span out[] = {{grad_x, p.T * d->C * es}, {grad_w, (size_t)d->O * d->C * es}, {ws, p.bwd}};
  if (int rc = block_spans(in, 2, out, 3, 1, nullptr, nullptr)) return rc;
  DeviceScope ds;
  if (int rc = ds.bind(h)) return rc;
  char* b = static_cast<char*>(ws);
  const char* k = static_cast<const char*>(saved);
  hipError_t e = dcn::launch_fp8_quantize(
      d->B, d->O, d->P, d->layout, d->dtype, grad_y, grad_x ? b + p.gq : nullptr,
      grad_x ? b + p.gs : nullptr, grad_w ? b + p.gc : nullptr, grad_w ? b + p.gcs : nullptr,
      ds.stream);
  const bool maps = d->layout == DCN_NCHW;
  if (e == hipSuccess && grad_x)
    e = dcn::launch_fp8_matmul(p.gx, maps ? k + p.wt : b + p.gq, maps ? k + p.wts : b + p.gs,
                               maps ? b + p.gq : k + p.wt, maps ? b + p.gs : k + p.wts, grad_x,
                               b + p.mmb, ds.stream);
  if (e == hipSuccess && grad_w)
    e = dcn::launch_fp8_matmul(p.gw, b + p.gc, b + p.gcs, k + p.xc, k + p.xcs, grad_w, b + p.mmb,
                               ds.stream);
  return done(e, "fp8_pointwise backward");
}

int dcn_fp8_quantize(dcn_handle* h, const dcn_fp8_desc* d, const void* v, void* q_tok, void* s_tok,
                     void* q_ch, void* s_ch) {
  if (!d) return fail(DCN_ERR_INVALID, "null descriptor");
  if (d->B <= 0 || d->C <= 0 || d->P <= 0) return fail(DCN_ERR_INVALID, "B, C, P must be positive");
  if (!dtype_ok(d->dtype)) return fail(DCN_ERR_INVALID, "unknown dtype");
  if (d->layout != DCN_NCHW && d->layout != DCN_NHWC) return fail(DCN_ERR_INVALID, "unknown layout");
  const bool maps = d->layout == DCN_NCHW;
  const size_t T = (size_t)d->B * d->P, C = d->C;
  const size_t kt = maps ? d->B * up128(d->P) : up128(T);
  if (T > (1u << 30) || kt > (1u << 30) || C > (1u << 30) ||
      !tiles_ok(maps ? d->C : (double)T, maps ? d->P : d->C, maps ? d->B : 1))
    return fail(DCN_ERR_UNSUPPORTED, "tensor too large");
  if (int rc = fp8_pair(q_tok, s_tok, "by token")) return rc;
  if (int rc = fp8_pair(q_ch, s_ch, "by channel")) return rc;
  if (!v || !(q_tok || q_ch)) return fail(DCN_ERR_INVALID, "null tensor");
  const size_t es = dtype_bytes(d->dtype);
  const Span in[] = {{v, T * C * es}};
  if (!aligned(v, es)) return fail(DCN_ERR_INVALID, "tensor not aligned to its elements");
  const Span out[] = {{q_tok, fp8_bytes(T, up128(C))}, {s_tok, exp_bytes(T, up128(C), 1)},
                      {q_ch, fp8_bytes(C, kt)}, {s_ch, exp_bytes(C, kt, 1)}};
  if (int rc = block_spans(in, 1, out, 4, 1, nullptr, nullptr)) return rc;
  DeviceScope ds;
  if (int rc = ds.bind(h)) return rc;
  return done(dcn::launch_fp8_quantize(d->B, d->C, d->P, d->layout, d->dtype, v, q_tok, s_tok, q_ch,
                                       s_ch, ds.stream),
              "fp8_quantize");
}

int dcn_fp8_quantize_weight(dcn_handle* h, int O, int C, int dtype, const void* w, void* q, void* s,
                            void* qT, void* sT) {
  if (O <= 0 || C <= 0) return fail(DCN_ERR_INVALID, "O, C must be positive");
  if (!dtype_ok(dtype)) return fail(DCN_ERR_INVALID, "unknown dtype");
  if (O > (1 << 30) || C > (1 << 30) || !tiles_ok(O, C, 1))
    return fail(DCN_ERR_UNSUPPORTED, "weight too large");
  if (int rc = fp8_pair(q, s, "weight")) return rc;
  if (int rc = fp8_pair(qT, sT, "transposed weight")) return rc;
  if (!w || !(q || qT)) return fail(DCN_ERR_INVALID, "null tensor");
  const size_t es = dtype_bytes(dtype);
  if (!aligned(w, es)) return fail(DCN_ERR_INVALID, "tensor not aligned to its elements");
  const Span in[] = {{w, (size_t)O * C * es}};
  const Span out[] = {{q, fp8_bytes(O, up128(C))}, {s, exp_bytes(O, up128(C), 128)},
                      {qT, fp8_bytes(C, up128(O))}, {sT, exp_bytes(C, up128(O), 128)}};
  if (int rc = block_spans(in, 1, out, 4, 1, nullptr, nullptr)) return rc;
  DeviceScope ds;
  if (int rc = ds.bind(h)) return rc;
  return done(dcn::launch_fp8_quantize_weight(O, C, dtype, w, q, s, qT, sT, ds.stream),
              "fp8_quantize_weight");
}

int dcn_fp8_matmul_workspace(const dcn_fp8_matmul_desc* d, size_t* bytes) {
  if (int rc = fp8_matmul_check(d)) return rc;
  if (!bytes) return fail(DCN_ERR_INVALID, "null out pointer");
  *bytes = dcn::fp8_matmul_ws_bytes(*d);
  return DCN_OK;
}

int dcn_fp8_matmul(dcn_handle* h, const dcn_fp8_matmul_desc* d, const void* a, const void* sa,
                   const void* b, const void* sb, void* out, void* ws, size_t ws_bytes) {
  if (int rc = fp8_matmul_check(d)) return rc;
  if (!a || !b || !out) return fail(DCN_ERR_INVALID, "null tensor");
  if (int rc = fp8_pair(a, sa, "a")) return rc;
  if (int rc = fp8_pair(b, sb, "b")) return rc;
  const size_t es = dtype_bytes(d->out_dtype), need = dcn::fp8_matmul_ws_bytes(*d);
  if (need && (!ws || ws_bytes < need))
    return fail(DCN_ERR_WORKSPACE, "fp8_matmul workspace too small");
  if (!aligned(ws, 256)) return fail(DCN_ERR_INVALID, "workspace must be 256-byte aligned");
  if (!aligned(out, es)) return fail(DCN_ERR_INVALID, "tensor not aligned to its elements");
  const Span in[] = {{a, fp8_bytes(d->M, d->K)}, {sa, exp_bytes(d->M, d->K, d->a_block)},
                     {b, fp8_bytes(d->N, d->K)}, {sb, exp_bytes(d->N, d->K, d->b_block)}};
  const Span outs[] = {{out, (size_t)d->M * d->N * es}, {need ? ws : nullptr, need}};
  if (int rc = block_spans(in, 4, outs, 2, 1, nullptr, nullptr)) return rc;
  DeviceScope ds;
  if (int rc = ds.bind(h)) return rc;
  return done(dcn::launch_fp8_matmul(*d, a, sa, b, sb, out, ws, ds.stream), "fp8_matmul");
}

int dcn_block_norm_fwd(dcn_handle* h, const dcn_block_desc* d, const dcn_block_io* io) {
  dcn::BlockArgs a;
  if (int rc = block_inputs(d, io, &a)) return rc;
  if ((io->y != nullptr) != (d->pre != DCN_NORM_NONE))
    return fail(DCN_ERR_INVALID, "y and the pre norm must come together");
  if (!io->x && io->out) return fail(DCN_ERR_INVALID, "without x there is no out");
  if (!io->y && !io->out) return fail(DCN_ERR_INVALID, "no output");
  a.out = io->out; a.y = io->y;
  const size_t es = dtype_bytes(d->dtype), full = (size_t)d->B * d->C * d->P * es,
               vec = (size_t)d->C * es;
  const size_t gate = d->gate == DCN_GATE_FULL ? full : (size_t)d->B * d->C * es;
  const Span in[] = {{io->x, full}, {io->residual, full}, {io->gate, gate}, {io->scale, vec},
                     {io->w_post, vec}, {io->b_post, vec}, {io->w_pre, vec}, {io->b_pre, vec},
                     {io->rng, 16}};
  const Span out[] = {{io->out, full}, {io->y, full}, {io->stats, (size_t)d->B * d->P * 16}};
  if (int rc = block_spans(in, 9, out, 3, es, io->out, io->residual)) return rc;
  DeviceScope ds;
  if (int rc = ds.bind(h)) return rc;
  return done(dcn::launch_block_norm_fwd(a, ds.stream), "block_norm forward");
}

int dcn_block_norm_workspace(const dcn_block_desc* d, size_t* bytes) {
  dcn::BlockArgs a;
  if (int rc = block_geo(d, &a)) return rc;
  if (!bytes) return fail(DCN_ERR_INVALID, "null out pointer");
  *bytes = dcn::block_norm_ws_floats(a) * sizeof(float);
  return DCN_OK;
}

int dcn_block_norm_bwd(dcn_handle* h, const dcn_block_desc* d, const dcn_block_io* io, void* ws,
                       size_t ws_bytes) {
  dcn::BlockArgs a;
  if (int rc = block_inputs(d, io, &a)) return rc;
  if (!io->grad_out && !io->grad_y) return fail(DCN_ERR_INVALID, "neither grad_out nor grad_y");
  if (io->grad_y && !d->pre) return fail(DCN_ERR_INVALID, "grad_y without a pre norm");
  if (!io->x && (io->grad_out || io->grad_x || io->grad_gate || io->grad_scale ||
                 io->grad_w_post || io->grad_b_post))
    return fail(DCN_ERR_INVALID, "without x there is no out and no gradient of the block");
  if (io->grad_gate && !d->gate) return fail(DCN_ERR_INVALID, "grad_gate without a gate");
  if ((io->grad_w_post || io->grad_b_post) && !d->post)
    return fail(DCN_ERR_INVALID, "grad_w_post / grad_b_post without a post norm");
  if ((io->grad_w_pre || io->grad_b_pre) && !d->pre)
    return fail(DCN_ERR_INVALID, "grad_w_pre / grad_b_pre without a pre norm");
  if (!(io->grad_x || io->grad_residual || io->grad_gate || io->grad_scale || io->grad_w_post ||
        io->grad_b_post || io->grad_w_pre || io->grad_b_pre))
    return fail(DCN_ERR_INVALID, "no gradient wanted");
  a.go = io->grad_out; a.gy = io->grad_y;
  a.gx = io->grad_x; a.gr = io->grad_residual; a.gg = io->grad_gate; a.gs = io->grad_scale;
  a.gw1 = io->grad_w_post; a.gb1 = io->grad_b_post; a.gw2 = io->grad_w_pre; a.gb2 = io->grad_b_pre;
  const size_t need = dcn::block_norm_ws_floats(a) * sizeof(float);
  if (!ws || ws_bytes < need) return fail(DCN_ERR_WORKSPACE, "block_norm workspace too small");
  if (!aligned(ws, 256)) return fail(DCN_ERR_INVALID, "workspace must be 256-byte aligned");
  const size_t es = dtype_bytes(d->dtype), full = (size_t)d->B * d->C * d->P * es,
               vec = (size_t)d->C * es;
  const size_t gate = d->gate == DCN_GATE_FULL ? full : (size_t)d->B * d->C * es;
  const Span in[] = {{io->x, full}, {io->residual, full}, {io->gate, gate}, {io->scale, vec},
                     {io->w_post, vec}, {io->b_post, vec}, {io->w_pre, vec}, {io->b_pre, vec},
                     {io->grad_out, full}, {io->grad_y, full}, {io->rng, 16},
                     {io->stats, (size_t)d->B * d->P * 16}};
  const Span out[] = {{io->grad_x, full}, {io->grad_residual, full}, {io->grad_gate, gate},
                      {io->grad_scale, vec}, {io->grad_w_post, vec}, {io->grad_b_post, vec},
                      {io->grad_w_pre, vec}, {io->grad_b_pre, vec}, {ws, need}};
  if (int rc = block_spans(in, 12, out, 9, es, nullptr, nullptr)) return rc;
  a.ws = static_cast<float*>(ws);
  DeviceScope ds;
  if (int rc = ds.bind(h)) return rc;
  return done(dcn::launch_block_norm_bwd(a, ds.stream), "block_norm backward");
}

int dcn_dropout_fwd(dcn_handle* h, const dcn_dropout_desc* d, const void* x, const void* residual,
                    void* y, const void* rng) {
  return dropout(h, d, x, residual, y, rng);
}

int dcn_dropout_bwd(dcn_handle* h, const dcn_dropout_desc* d, const void* grad_y, void* grad_x,
                    const void* rng) {
  return dropout(h, d, grad_y, nullptr, grad_x, rng);
}

}  // extern "C"
