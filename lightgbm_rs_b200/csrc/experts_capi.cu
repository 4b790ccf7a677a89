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

bool is_act(int32_t act) {
  return act == LGBM_B200_ACT_NONE || act == LGBM_B200_ACT_RELU || act == LGBM_B200_ACT_SILU ||
         act == LGBM_B200_ACT_GELU;
}

// The weight rows of a gated layer, or -1 where its width is refused anyway.
int32_t gated_outer(int32_t hidden) {
  return hidden < 1 || hidden > kMaxWidth / 2 ? -1 : 2 * hidden;
}
int check_hidden(const char* what, int32_t hidden) {
  if (hidden < 1) return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: hidden %d", what, hidden);
  if (hidden > kMaxWidth / 2)
    return refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, "%s: hidden %d (at most %d)", what, hidden,
                  kMaxWidth / 2);
  return LGBM_B200_OK;
}

int check_epilogue(const char* what, const MatmulCall& c) {
  const Epilogue& e = c.epilogue;
  if (!is_act(e.act)) return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: activation %d", what, e.act);
  if (e.residual && e.residual_pitch < c.outer)
    return refuse(LGBM_B200_LENGTH_MISMATCH, "%s: residual pitch %lld < outer %d", what,
                  (long long)e.residual_pitch, c.outer);
  if (!aligned32(e.pre))
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: pre is not 32-byte aligned", what);
  return check_starts(what, {{e.bias, 2}, {e.residual, 2}});
}

int run_product(const char* what, const MatmulCall& c, void* workspace, int64_t workspace_bytes,
                void* stream) {
  if (int rc = check_product(what, c)) return rc;
  if (c.epilogue.on)
    if (int rc = check_epilogue(what, c)) return rc;
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

// The gradient of what the activation was given, in the workspace ahead of what the products need.
int64_t dpre_pitch(int32_t outer) { return ((int64_t)outer + 7) / 8 * 8; }
int64_t dpre_bytes(int64_t rows, int32_t outer) {
  return (rows * dpre_pitch(outer) * 2 + 255) / 256 * 256;
}
int64_t sums_bytes(int64_t rows, int32_t experts, int32_t outer) {
  return (linear_grad_workspace(rows, experts, outer) + 255) / 256 * 256;
}

// Both gradients of a layer's products and what comes before them; c.dy, c.outer are the layer's.
int run_layer_backward(const char* what, MatmulCall c, bool gated, int32_t act, const void* pre,
                       void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!is_act(act)) return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: activation %d", what, act);
  if (!c.dx && !c.dw && !dbias && c.rows > 0)
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: no gradient is wanted", what);
  if ((c.dw || dbias) && c.grad_dtype != c.dtype && c.grad_dtype != LGBM_B200_DTYPE_F32)
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: dtype %d of the weights' gradients", what,
                  c.grad_dtype);
  const int32_t width = gated ? c.outer / 2 : c.outer;  // of dy
  const bool turns = gated || act != LGBM_B200_ACT_NONE;  // dpre is not dy itself
  // what check_product sees of dy: a pitch that fits, where dpre takes its place
  MatmulCall p = c;
  p.layer = true;
  if (turns) p.dy_pitch = dpre_pitch(c.outer);
  if (int rc = check_product(what, p)) return rc;
  if (c.dy_pitch < width)
    return refuse(LGBM_B200_LENGTH_MISMATCH, "%s: dy pitch %lld < %d", what,
                  (long long)c.dy_pitch, width);
  if (c.rows > 0 && (!c.dy || (turns && !pre)))
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  if (turns && !aligned32(pre))
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: pre is not 32-byte aligned", what);
  if (int rc = check_starts(what, {{c.dy, 2}, {dbias, dbias ? elem_size(c.grad_dtype) : 1}}))
    return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (c.rows == 0) {
    cudaError_t err = cudaSuccess;
    const int64_t size = elem_size(c.grad_dtype);
    if (c.dw)
      err = cudaMemsetAsync(c.dw, 0, (size_t)(size * c.experts * c.outer * c.inner), st);
    if (err == cudaSuccess && dbias)
      err = cudaMemsetAsync(dbias, 0, (size_t)(size * c.experts * c.outer), st);
    return launched(err, what);
  }
  char* ws = static_cast<char*>(workspace);
  int64_t need = 0;
  if (turns) {
    p.dy = ws;
    need += dpre_bytes(c.rows, c.outer);
  }
  float* sums = reinterpret_cast<float*>(ws + need);
  if (dbias) need += sums_bytes(c.rows, c.experts, c.outer);
  const bool products = c.dx || c.dw;
  const int64_t own = need;
  if (turns) p.dy = reinterpret_cast<const void*>((uintptr_t)256);  // aligned, for the question
  if (products) need += matmul_workspace(p);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned16(workspace))))
    return refuse(LGBM_B200_LENGTH_MISMATCH, "%s: workspace of %lld bytes, %lld are needed",
                  what, (long long)workspace_bytes, (long long)need);
  if (turns) p.dy = ws;
  if (gated) {
    if (int rc = launched(launch_gated_grad(c.dy, c.dy_pitch, pre, c.dtype, act, c.rows, width, ws,
                                            p.dy_pitch, st),
                          what))
      return rc;
  } else if (turns || dbias) {
    LinearGrad l{};
    l.dy = c.dy;
    l.dy_pitch = c.dy_pitch;
    l.pre = pre;
    l.dtype = c.dtype;
    l.grad_dtype = c.grad_dtype;
    l.act = act;
    l.offsets = c.offsets;
    l.rows = c.rows;
    l.experts = c.experts;
    l.outer = c.outer;
    l.dpre = turns ? ws : nullptr;
    l.dpre_pitch = p.dy_pitch;
    l.dbias = dbias;
    l.sums = sums;
    if (int rc = launched(launch_linear_grad(l, st), what)) return rc;
  }
  return products ? launched(launch_matmul(p, ws + own, st), what) : LGBM_B200_OK;
}

int64_t layer_backward_workspace(const void* dy, int64_t dy_pitch, const void* x, int64_t x_pitch,
                                 const int32_t* index, const void* w, int32_t act, bool gated,
                                 int64_t rows, int32_t experts, int32_t inner, int32_t outer,
                                 int32_t want_dx, int32_t want_dw, int32_t want_dbias) {
  if (rows < 1 || experts < 1 || inner < 1 || outer < 1) return 0;
  const bool turns = gated || act != LGBM_B200_ACT_NONE;
  int64_t need = (turns ? dpre_bytes(rows, outer) : 0) +
                 (want_dbias ? sums_bytes(rows, experts, outer) : 0);
  MatmulCall c{};
  c.x = x;
  c.x_pitch = x_pitch;
  c.index = index;
  c.dy = turns ? reinterpret_cast<const void*>((uintptr_t)256) : dy;
  c.dy_pitch = turns ? dpre_pitch(outer) : dy_pitch;
  c.w = w;
  c.rows = rows;
  c.experts = experts;
  c.inner = inner;
  c.outer = outer;
  c.dx = want_dx ? &c : nullptr;  // wanted; not written here
  c.dw = want_dw ? &c : nullptr;
  c.layer = true;
  return c.dx || c.dw ? need + matmul_workspace(c) : need;
}

// Bytes of all tensors of a norm: their windows are counted in 32 bits.
constexpr int64_t kMaxNormBytes = 1ll << 44;

int run_norm(const char* what, const lgbm_b200_experts_tensor* tensors, int64_t count, bool scale,
             double max_norm, float* norm, void* workspace, int64_t workspace_bytes,
             void* stream) {
  if (count < 0 || (count > 0 && !tensors) || !norm)
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: %lld tensors, or a null argument", what,
                  (long long)count);
  if (count > (1 << 24))
    return refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, "%s: %lld tensors (at most %d)", what,
                  (long long)count, 1 << 24);
  if (scale && !(max_norm >= 0.0))
    return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: max_norm %g", what, max_norm);
  if (int rc = check_starts(what, {{norm, 4}})) return rc;
  int64_t left = kMaxNormBytes - count * 65536;  // a window of each may be nearly empty
  for (int64_t i = 0; i < count; ++i) {
    const lgbm_b200_experts_tensor& t = tensors[i];
    if (!is_float(t.dtype) || t.count < 0 ||
        (t.count > 0 && (!t.in || (scale && !t.out))))
      return refuse(LGBM_B200_INVALID_ARGUMENT,
                    "%s: tensor %lld: dtype %d, %lld elements, or a null argument", what,
                    (long long)i, t.dtype, (long long)t.count);
    const int size = elem_size(t.dtype);
    // (no division a tensor: those of 1021 took the host 5 us)
    if (t.count > left >> (size == 4 ? 2 : 1))
      return refuse(LGBM_B200_CAPABILITY_UNAVAILABLE, "%s: more than %lld bytes", what,
                    (long long)kMaxNormBytes);
    left -= t.count * size;
    const void* const out = scale ? t.out : nullptr;
    if (t.count > 0 &&
        ((reinterpret_cast<uintptr_t>(t.in) | reinterpret_cast<uintptr_t>(out)) & (size - 1)))
      if (int rc = check_starts(what, {{t.in, size}, {out, size}})) return rc;
  }
  const int64_t need = norm_workspace(tensors, count);
  if (workspace_bytes < need || (need > 0 && (!workspace || !aligned16(workspace))))
    return refuse(LGBM_B200_LENGTH_MISMATCH, "%s: workspace of %lld bytes, %lld are needed",
                  what, (long long)workspace_bytes, (long long)need);
  const NormCall c{tensors, count, scale, max_norm, workspace, norm};
  return launched(launch_norm(c, reinterpret_cast<cudaStream_t>(stream)), what);
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

int64_t lgbm_b200_experts_linear_workspace(const void* x, int64_t x_pitch, const int32_t* index,
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
  c.epilogue.on = true;
  return matmul_workspace(c);
}

int lgbm_b200_experts_linear(const void* x, int64_t x_rows, int64_t x_pitch,
                             const int32_t* index, const void* w, const void* bias,
                             const void* residual, int64_t residual_pitch, const int32_t* offsets,
                             int32_t dtype, int32_t act, int64_t rows, int32_t experts,
                             int32_t inner, int32_t outer, void* y, void* pre, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  const char* what = "experts_linear";
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
  c.epilogue = {true, false, act, bias, residual, residual_pitch, pre};
  return run_product(what, c, workspace, workspace_bytes, stream);
}

int lgbm_b200_experts_gated(const void* x, int64_t x_rows, int64_t x_pitch, const int32_t* index,
                            const void* w, const int32_t* offsets, int32_t dtype, int32_t act,
                            int64_t rows, int32_t experts, int32_t inner, int32_t hidden, void* h,
                            void* pre, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "experts_gated";
  if (!h && rows > 0) return refuse(LGBM_B200_INVALID_ARGUMENT, "%s: null argument", what);
  if (int rc = check_hidden(what, hidden)) return rc;
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
  c.outer = gated_outer(hidden);
  c.y = h ? h : &c;  // no rows: nothing is written
  c.epilogue = {true, true, act, nullptr, nullptr, 0, pre};
  return run_product(what, c, workspace, workspace_bytes, stream);
}

int64_t lgbm_b200_experts_linear_backward_workspace(
    const void* dy, int64_t dy_pitch, const void* x, int64_t x_pitch, const int32_t* index,
    const void* w, int32_t act, int64_t rows, int32_t experts, int32_t inner, int32_t outer,
    int32_t want_dx, int32_t want_dw, int32_t want_dbias) {
  return layer_backward_workspace(dy, dy_pitch, x, x_pitch, index, w, act, false, rows, experts,
                                  inner, outer, want_dx, want_dw, want_dbias);
}

int lgbm_b200_experts_linear_backward(const void* dy, int64_t dy_pitch, const void* pre,
                                      const void* x, int64_t x_rows, int64_t x_pitch,
                                      const int32_t* index, const void* w, const int32_t* offsets,
                                      int32_t dtype, int32_t grad_dtype, int32_t act, int64_t rows,
                                      int32_t experts, int32_t inner, int32_t outer, void* dx,
                                      void* dw, void* dbias, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
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
  return run_layer_backward("experts_linear_backward", c, false, act, pre, dbias, workspace,
                            workspace_bytes, stream);
}

int64_t lgbm_b200_experts_gated_backward_workspace(const void* x, int64_t x_pitch,
                                                   const int32_t* index, const void* w,
                                                   int64_t rows, int32_t experts, int32_t inner,
                                                   int32_t hidden, int32_t want_dx,
                                                   int32_t want_dw) {
  return layer_backward_workspace(nullptr, 0, x, x_pitch, index, w, LGBM_B200_ACT_NONE, true, rows,
                                  experts, inner, gated_outer(hidden), want_dx, want_dw, 0);
}

int lgbm_b200_experts_gated_backward(const void* dh, int64_t dh_pitch, const void* pre,
                                     const void* x, int64_t x_rows, int64_t x_pitch,
                                     const int32_t* index, const void* w, const int32_t* offsets,
                                     int32_t dtype, int32_t grad_dtype, int32_t act, int64_t rows,
                                     int32_t experts, int32_t inner, int32_t hidden, void* dx,
                                     void* dw, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  const char* what = "experts_gated_backward";
  if (int rc = check_hidden(what, hidden)) return rc;
  MatmulCall c{};
  c.dtype = dtype;
  c.grad_dtype = grad_dtype;
  c.x = x;
  c.x_rows = x_rows;
  c.x_pitch = x_pitch;
  c.index = index;
  c.dy = dh;
  c.dy_pitch = dh_pitch;
  c.w = w;
  c.offsets = offsets;
  c.rows = rows;
  c.experts = experts;
  c.inner = inner;
  c.outer = gated_outer(hidden);
  c.dx = dx;
  c.dw = dw;
  return run_layer_backward(what, c, true, act, pre, nullptr, workspace, workspace_bytes, stream);
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

int64_t lgbm_b200_experts_norm_workspace(const lgbm_b200_experts_tensor* tensors, int64_t count) {
  return count < 1 || !tensors ? 0 : norm_workspace(tensors, count);
}

int lgbm_b200_experts_grad_norm(const lgbm_b200_experts_tensor* tensors, int64_t count,
                                float* norm, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  return run_norm("experts_grad_norm", tensors, count, false, 0.0, norm, workspace,
                  workspace_bytes, stream);
}

int lgbm_b200_experts_clip_grads(const lgbm_b200_experts_tensor* tensors, int64_t count,
                                 double max_norm, float* norm, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  return run_norm("experts_clip_grads", tensors, count, true, max_norm, norm, workspace,
                  workspace_bytes, stream);
}

int lgbm_b200_experts_errors(uint32_t* bits_out) {
  if (!bits_out) return refuse(LGBM_B200_INVALID_ARGUMENT, "experts_errors: null argument");
  return launched(take_matmul_errors(bits_out), "experts_errors");
}

}  // extern "C"
