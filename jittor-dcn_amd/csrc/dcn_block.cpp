// dcn_block.cpp — entry points of the residual block's operators (include/dcn.h): argument
// checks, then one launcher each. Nothing here allocates, synchronises or keeps state, so every
// call can be captured into a graph.
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

}  // namespace

extern "C" {

int dcn_dropout_fwd(dcn_handle* h, const dcn_dropout_desc* d, const void* x, const void* residual,
                    void* y, const void* rng) {
  return dropout(h, d, x, residual, y, rng);
}

int dcn_dropout_bwd(dcn_handle* h, const dcn_dropout_desc* d, const void* grad_y, void* grad_x,
                    const void* rng) {
  return dropout(h, d, grad_y, nullptr, grad_x, rng);
}

}  // extern "C"
