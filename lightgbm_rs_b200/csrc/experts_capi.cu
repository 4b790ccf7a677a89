// C entry points of the expert-layer operators: argument checks, then the launches. Nothing
// here allocates or throws, and nothing but lgbm_b200_experts_errors waits for the device.
#include <cstdarg>
#include <cstdio>
#include <initializer_list>

#include "experts.cuh"

using namespace lgbm_b200;
using namespace lgbm_b200::experts;

namespace {

int refuse(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_last_error(code, buf);
}

int launched(cudaError_t err, const char* what) {
  if (err == cudaSuccess) return LGBM_B200_OK;
  cudaGetLastError();  // not sticky: reported here
  if (err == cudaErrorNoDevice || err == cudaErrorInsufficientDriver)
    return refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, "%s: no CUDA device", what);
  return refuse(LGBM_B200_RUNTIME, "%s failed: %s", what, cudaGetErrorString(err));
}

bool is_float(int32_t dtype) {
  return dtype == LGBM_B200_DTYPE_F32 || dtype == LGBM_B200_DTYPE_BF16 ||
         dtype == LGBM_B200_DTYPE_F16;
}

struct Array {
  const void* p;
  int size;  // bytes of an element
};

// An access off its element's size faults on the device. Null starts everywhere.
int check_starts(const char* what, std::initializer_list<Array> arrays) {
  int i = 0;
  for (const Array& a : arrays) {
    if (reinterpret_cast<uintptr_t>(a.p) % a.size != 0)
      return refuse(LGBM_B200_INVALID_ARGUMENT,
                    "%s: array %d at %p does not start at a multiple of its %d-byte elements", what,
                    i, a.p, a.size);
    ++i;
  }
  return LGBM_B200_OK;
}

// Grouped rows are counted in 32 bits, with room for a tile past the last one.
constexpr int64_t kMaxRows = 0x7FFFFFFFll - 65536;
// Bytes of a row of a product's operand are counted in 32 bits.
constexpr int32_t kMaxWidth = 1 << 28;

int check_gate(const char* what, int32_t dtype, int64_t tokens, int32_t experts, int64_t pitch,
               int32_t k) {
  if (!is_float(dtype)) return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: dtype %d", what, dtype);
  if (tokens < 0 || experts < 1 || k < 1 || k > experts || pitch < experts)
    return refuse(LGBM_B200_INVALID_ARGUMENT,
                  "%s: tokens %lld, experts %d, k %d, pitch %lld: want tokens >= 0, "
                  "1 <= k <= experts <= pitch",
                  what, (long long)tokens, experts, k, (long long)pitch);
  if (experts > kMaxExperts || k > kMaxChosen || tokens > kMaxRows / k)
    return refuse(LGBM_B200_CAPABILITY_UNAVAILABLE,
                  "%s: %d experts (at most %d), k %d (at most %d), %lld rows (at most %lld)",
                  what, experts, kMaxExperts, k, kMaxChosen, (long long)tokens * k,
                  (long long)kMaxRows);
  return LGBM_B200_OK;
}

int check_product(const char* what, const MatmulCall& c) {
  if (c.dtype != LGBM_B200_DTYPE_BF16 && c.dtype != LGBM_B200_DTYPE_F16)
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: dtype %d is not bf16 or f16", what, c.dtype);
  if (c.dw && c.grad_dtype != c.dtype && c.grad_dtype != LGBM_B200_DTYPE_F32)
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: dw's dtype %d", what, c.grad_dtype);
  if (c.rows < 0 || c.experts < 1 || c.inner < 1 || c.outer < 1)
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: rows %lld, experts %d, inner %d, outer %d",
                  what, (long long)c.rows, c.experts, c.inner, c.outer);
  if (c.experts > kMaxExperts || c.rows > kMaxRows || c.x_rows > kMaxRows ||
      c.inner > kMaxWidth || c.outer > kMaxWidth)
    return refuse(LGBM_B200_CAPABILITY_UNAVAILABLE,
                  "%s: %d experts (at most %d), %lld rows of %lld (at most %lld), inner %d and "
                  "outer %d (at most %d)",
                  what, c.experts, kMaxExperts, (long long)c.rows, (long long)c.x_rows,
                  (long long)kMaxRows, c.inner, c.outer, kMaxWidth);
  const bool reads_x = c.y || c.dw, reads_dy = c.dx || c.dw, reads_w = c.y || c.dx;
  if (!c.offsets || (c.rows > 0 && ((reads_x && !c.x) || (reads_dy && !c.dy))) ||
      (reads_w && !c.w))
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  if (int rc = check_starts(what, {{reads_x ? c.x : nullptr, 2},
                                   {reads_dy ? c.dy : nullptr, 2},
                                   {reads_w ? c.w : nullptr, 2},
                                   {reads_x ? c.index : nullptr, 4},
                                   {c.offsets, 4},
                                   {c.y, 2},
                                   {c.dx, 2},
                                   {c.dw, c.dw ? elem_size(c.grad_dtype) : 1}}))
    return rc;
  if (reads_x && (c.x_pitch < c.inner || c.x_rows < (c.rows > 0) ||
                  (!c.index && c.x_rows != c.rows)))
    return refuse(LGBM_B200_LENGTH_MISMATCH,
                  "%s: x has %lld rows of pitch %lld, want %lld of at least %d", what,
                  (long long)c.x_rows, (long long)c.x_pitch, (long long)c.rows, c.inner);
  if (reads_dy && c.dy_pitch < c.outer)
    return refuse(LGBM_B200_LENGTH_MISMATCH, "%s: dy pitch %lld < outer %d", what,
                  (long long)c.dy_pitch, c.outer);
  return LGBM_B200_OK;
}

int run_product(const char* what, const MatmulCall& c, void* workspace, int64_t workspace_bytes,
                void* stream) {
  if (int rc = check_product(what, c)) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (c.rows == 0) {
    if (!c.dw) return LGBM_B200_OK;
    return launched(
        cudaMemsetAsync(c.dw, 0, (size_t)c.experts * c.outer * c.inner * elem_size(c.grad_dtype),
                        st),
        what);
  }
  const int64_t need = matmul_workspace(c);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned16(workspace))))
    return refuse(LGBM_B200_LENGTH_MISMATCH, "%s: workspace of %lld bytes, %lld are needed",
                  what, (long long)workspace_bytes, (long long)need);
  return launched(launch_matmul(c, workspace, st), what);
}

}  // namespace

extern "C" {

int64_t lgbm_b200_experts_route_workspace(int64_t tokens, int32_t experts, int32_t k) {
  if (tokens < 0 || experts < 1 || experts > kMaxExperts || k < 1) return 0;
  return route_workspace(tokens, experts, k);
}

int lgbm_b200_experts_route(const void* logits, int32_t dtype, int64_t tokens, int32_t experts,
                            int64_t pitch, int32_t k, int32_t normalize, float* weights,
                            int32_t* chosen, int32_t* position, int32_t* rows, int32_t* offsets,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "experts_route";
  if (int rc = check_gate(what, dtype, tokens, experts, pitch, k)) return rc;
  if (!offsets || (tokens > 0 && (!logits || !weights || !chosen || !position || !rows)))
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  if (int rc = check_starts(what, {{logits, elem_size(dtype)},
                                   {weights, 4},
                                   {chosen, 4},
                                   {position, 4},
                                   {rows, 4},
                                   {offsets, 4}}))
    return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (tokens == 0)
    return launched(cudaMemsetAsync(offsets, 0, sizeof(int32_t) * (experts + 1), st), what);
  const int64_t need = route_workspace(tokens, experts, k);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned16(workspace))))
    return refuse(LGBM_B200_LENGTH_MISMATCH, "%s: workspace of %lld bytes, %lld are needed",
                  what, (long long)workspace_bytes, (long long)need);
  return launched(launch_route(logits, dtype, tokens, experts, pitch, k, normalize != 0, weights,
                               chosen, position, rows, offsets, workspace, st),
                  what);
}

int lgbm_b200_experts_route_backward(const float* dweights, const float* weights,
                                     const int32_t* chosen, const void* logits, int32_t dtype,
                                     int64_t tokens, int32_t experts, int64_t pitch, int32_t k,
                                     int32_t normalize, void* dlogits, void* stream) {
  const char* what = "experts_route_backward";
  if (int rc = check_gate(what, dtype, tokens, experts, pitch, k)) return rc;
  if (tokens == 0) return LGBM_B200_OK;
  if (!dweights || !weights || !chosen || !logits || !dlogits)
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  if (int rc = check_starts(what, {{dweights, 4},
                                   {weights, 4},
                                   {chosen, 4},
                                   {logits, elem_size(dtype)},
                                   {dlogits, elem_size(dtype)}}))
    return rc;
  return launched(launch_route_backward(dweights, weights, chosen, logits, dtype, tokens, experts,
                                        pitch, k, normalize != 0, dlogits,
                                        reinterpret_cast<cudaStream_t>(stream)),
                  what);
}

int lgbm_b200_experts_combine(const void* y, int32_t dtype, int64_t rows, int32_t width,
                              int64_t pitch, const int32_t* position, const float* weights,
                              int64_t tokens, int32_t k, void* out, void* stream) {
  const char* what = "experts_combine";
  if (!is_float(dtype) || rows < 0 || tokens < 0 || k < 1 || width < 1 || pitch < width)
    return refuse(LGBM_B200_INVALID_ARGUMENT,
                  "%s: dtype %d, rows %lld, width %d, pitch %lld, tokens %lld, k %d", what, dtype,
                  (long long)rows, width, (long long)pitch, (long long)tokens, k);
  if (tokens > kMaxRows || rows > kMaxRows)
    return refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, "%s: more than %lld rows", what,
                  (long long)kMaxRows);
  if (tokens == 0) return LGBM_B200_OK;
  if (!position || !out || (rows > 0 && !y))
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  if (int rc = check_starts(what, {{y, elem_size(dtype)},
                                   {position, 4},
                                   {weights, 4},
                                   {out, elem_size(dtype)}}))
    return rc;
  return launched(launch_combine(y, dtype, rows, width, pitch, position, weights, tokens, k, out,
                                 reinterpret_cast<cudaStream_t>(stream)),
                  what);
}

int lgbm_b200_experts_combine_backward(const void* dout, const void* y, int32_t dtype,
                                       int64_t rows, int32_t width, int64_t dout_pitch,
                                       int64_t pitch, const int32_t* position,
                                       const float* weights, int64_t tokens, int32_t k, void* dy,
                                       float* dweights, void* stream) {
  const char* what = "experts_combine_backward";
  if (!is_float(dtype) || tokens < 0 || k < 1 || width < 1 || pitch < width ||
      dout_pitch < width)
    return refuse(LGBM_B200_INVALID_ARGUMENT,
                  "%s: dtype %d, width %d, pitches %lld and %lld, tokens %lld, k %d", what, dtype,
                  width, (long long)dout_pitch, (long long)pitch, (long long)tokens, k);
  if (tokens > kMaxRows / k)
    return refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, "%s: more than %lld rows", what,
                  (long long)kMaxRows);
  if (rows != tokens * k)
    return refuse(LGBM_B200_LENGTH_MISMATCH, "%s: %lld rows, want tokens * k = %lld", what,
                  (long long)rows, (long long)(tokens * k));
  if (tokens == 0) return LGBM_B200_OK;
  if (!dout || !position || !dy || (dweights && !y))
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  if (int rc = check_starts(what, {{dout, elem_size(dtype)},
                                   {dweights ? y : nullptr, elem_size(dtype)},
                                   {position, 4},
                                   {weights, 4},
                                   {dy, elem_size(dtype)},
                                   {dweights, 4}}))
    return rc;
  return launched(launch_combine_backward(dout, y, dtype, rows, width, dout_pitch, pitch,
                                          position, weights, tokens, k, dy, dweights,
                                          reinterpret_cast<cudaStream_t>(stream)),
                  what);
}

int lgbm_b200_experts_dropout(const void* x, const void* residual, int32_t dtype, int64_t rows,
                              int64_t width, int64_t pitch, int64_t residual_pitch, double p,
                              uint64_t seed, uint64_t offset, void* out, void* stream) {
  const char* what = "experts_dropout";
  if (!is_float(dtype) || rows < 0 || width < 0 || pitch < width ||
      (residual && residual_pitch < width) || (width > 0 && rows > INT64_MAX / 8 / width))
    return refuse(LGBM_B200_INVALID_ARGUMENT,
                  "%s: dtype %d, rows %lld, width %lld, pitches %lld and %lld", what, dtype,
                  (long long)rows, (long long)width, (long long)pitch,
                  (long long)residual_pitch);
  if (!(p >= 0.0 && p <= 1.0))
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: p %g is not in [0, 1]", what, p);
  if (rows == 0 || width == 0) return LGBM_B200_OK;
  if (!x || !out) return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  if (int rc = check_starts(what, {{x, elem_size(dtype)},
                                   {residual, elem_size(dtype)},
                                   {out, elem_size(dtype)}}))
    return rc;
  const uint32_t drop = (uint32_t)(p * 65536.0 + 0.5);
  return launched(launch_dropout(x, residual, dtype, rows, width, pitch, residual_pitch, drop,
                                 seed, offset, out, reinterpret_cast<cudaStream_t>(stream)),
                  what);
}

int64_t lgbm_b200_experts_matmul_workspace(const void* x, int64_t x_pitch, const int32_t* index,
                                           const void* w, int64_t rows, int32_t experts,
                                           int32_t inner, int32_t outer) {
  if (rows < 1 || experts < 1 || inner < 1 || outer < 1) return 0;
  MatmulCall c{};
  c.x = x;
  c.x_pitch = x_pitch;
  c.index = index;
  c.w = w;
  c.rows = rows;
  c.experts = experts;
  c.inner = inner;
  c.outer = outer;
  c.y = &c;  // wanted; not written here
  return matmul_workspace(c);
}

int lgbm_b200_experts_matmul(const void* x, int64_t x_rows, int64_t x_pitch,
                             const int32_t* index, const void* w, const int32_t* offsets,
                             int32_t dtype, int64_t rows, int32_t experts, int32_t inner,
                             int32_t outer, void* y, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  const char* what = "experts_matmul";
  if (!y && rows > 0) return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  MatmulCall c{};
  c.dtype = dtype;
  c.x = x;
  c.x_rows = x_rows;
  c.x_pitch = x_pitch;
  c.index = index;
  c.w = w;
  c.offsets = offsets;
  c.rows = rows;
  c.experts = experts;
  c.inner = inner;
  c.outer = outer;
  c.y = y ? y : &c;  // no rows: nothing is written
  return run_product(what, c, workspace, workspace_bytes, stream);
}

int64_t lgbm_b200_experts_matmul_backward_workspace(const void* dy, int64_t dy_pitch,
                                                    const void* x, int64_t x_pitch,
                                                    const int32_t* index, const void* w,
                                                    int64_t rows, int32_t experts, int32_t inner,
                                                    int32_t outer, int32_t want_dx,
                                                    int32_t want_dw) {
  if (rows < 1 || experts < 1 || inner < 1 || outer < 1) return 0;
  MatmulCall c{};
  c.x = x;
  c.x_pitch = x_pitch;
  c.index = index;
  c.dy = dy;
  c.dy_pitch = dy_pitch;
  c.w = w;
  c.rows = rows;
  c.experts = experts;
  c.inner = inner;
  c.outer = outer;
  c.dx = want_dx ? &c : nullptr;  // wanted; not written here
  c.dw = want_dw ? &c : nullptr;
  return matmul_workspace(c);
}

int lgbm_b200_experts_matmul_backward(const void* dy, int64_t dy_pitch, const void* x,
                                      int64_t x_rows, int64_t x_pitch, const int32_t* index,
                                      const void* w, const int32_t* offsets, int32_t dtype,
                                      int32_t grad_dtype, int64_t rows, int32_t experts,
                                      int32_t inner, int32_t outer, void* dx, void* dw,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "experts_matmul_backward";
  if (!dx && !dw && rows > 0)
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: neither dx nor dw is wanted", what);
  MatmulCall c{};
  c.dtype = dtype;
  c.grad_dtype = grad_dtype;
  c.x = x;
  c.x_rows = x_rows;
  c.x_pitch = x_pitch;
  c.index = index;
  c.dy = dy;
  c.dy_pitch = dy_pitch;
  c.w = w;
  c.offsets = offsets;
  c.rows = rows;
  c.experts = experts;
  c.inner = inner;
  c.outer = outer;
  c.dx = dx;
  c.dw = dw;
  return run_product(what, c, workspace, workspace_bytes, stream);
}

int lgbm_b200_experts_matmul_w4(const void* x, int64_t x_rows, int64_t x_pitch,
                                const int32_t* index, const uint8_t* q, const void* scales,
                                const uint8_t* zeros, int32_t group_size,
                                const int32_t* offsets, int32_t dtype, int64_t rows,
                                int32_t experts, int32_t inner, int32_t outer, void* y,
                                void* stream) {
  const char* what = "experts_matmul_w4";
  if (!y && rows > 0) return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  MatmulCall c{};
  c.dtype = dtype;
  c.x = x;
  c.x_rows = x_rows;
  c.x_pitch = x_pitch;
  c.index = index;
  c.w = q;
  c.offsets = offsets;
  c.rows = rows;
  c.experts = experts;
  c.inner = inner;
  c.outer = outer;
  c.y = y ? y : &c;  // no rows: nothing is written
  if (int rc = check_product(what, c)) return rc;
  if (group_size != 32 && group_size != 64 && group_size != 128)
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: group size %d is not 32, 64 or 128", what,
                  group_size);
  if (!scales) return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  if (!aligned16(q))
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: weights are not 16-byte aligned", what);
  if (int rc = check_starts(what, {{scales, 2}})) return rc;
  if (rows == 0) return LGBM_B200_OK;
  FewCall f{dtype, x,      x_rows, x_pitch, index, q,     group_size, scales,
            zeros, offsets, rows,   experts, inner, outer, y};
  return launched(launch_few(f, reinterpret_cast<cudaStream_t>(stream)), what);
}

int lgbm_b200_experts_errors(uint32_t* bits_out) {
  if (!bits_out) return refuse(LGBM_B200_INVALID_ARGUMENT, "experts_errors: null argument");
  return launched(take_matmul_errors(bits_out), "experts_errors");
}

}  // extern "C"
