// C entry points of the operators that serve dense networks token by token:
// norm, 4-bit dense layer, token log probabilities (include/b200_edsl.h).
// Argument checks only; none of these calls uses scratch memory.
#include <cmath>
#include <cstdint>
#include <string>
#include "../../include/b200_edsl.h"
#include "kernels.h"

using namespace b200;

namespace {

int bad(const char* msg) { return report_error(kErrInvalidArg, msg); }

int done(int rc, const char* what) {
  if (rc == kOk) return report_ok();
  if (rc == kErrTooLarge) return report_error(rc, (std::string(what) + ": too many rows").c_str());
  return report_error(rc, (std::string(what) + " launch failed: " + launch_error_text()).c_str());
}

bool plain_type(int dtype) { return dtype == kF32 || dtype == kBF16 || dtype == kF16; }
int64_t type_bytes(int dtype) { return dtype == kF32 ? 4 : dtype == kE4M3 ? 1 : 2; }

// An element type's buffer starts on a multiple of its size.
bool misplaced(const void* p, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % (uintptr_t)type_bytes(dtype) != 0;
}

constexpr int64_t kMaxIndex = (int64_t)1 << 31;

// K, N, group and type of packed 4-bit weights.
const char* w4_shape_error(int64_t K, int64_t N, int group, int s_dtype) {
  if (K < 0 || N < 0) return "negative dimension";
  if (K > kMaxIndex - 64 || N > kMaxIndex - 64) return "dimension exceeds the supported range";
  if (group != 32 && (group <= 0 || group % 64 != 0))
    return "group must be 32 or a multiple of 64";
  if (!plain_type(s_dtype)) return "scales must be f32, bf16 or f16";
  return nullptr;
}

W4Layout w4_layout(int64_t K, int64_t N, int group, int s_dtype, int has_zeros) {
  W4Layout w;
  w.K = K;
  w.N = N;
  w.group = group;
  w.s_dtype = s_dtype;
  w.has_zeros = has_zeros != 0;
  return w;
}

bool unaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace

extern "C" {

int b200_rms_norm(const void* X, int64_t ldx, const void* R, int64_t ldr, int dtype, const void* w,
                  int w_dtype, float eps, void* H, int64_t ldh, void* Y, int64_t ldy, int y_dtype,
                  float* scales, int64_t ld_scales, int group, int64_t M, int64_t N,
                  void* stream) {
  if (M < 0 || N < 0) return bad("negative dimension");
  if (M >= kMaxIndex || N >= kMaxIndex)
    return report_error(kErrTooLarge, "dimension exceeds the supported range");
  if (!plain_type(dtype)) return bad("X must be f32, bf16 or f16");
  if (w && w_dtype != dtype && w_dtype != kF32) return bad("w must be f32 or of X's type");
  if (!(eps > 0.0f) || std::isinf(eps)) return bad("eps must be positive and finite");
  if (y_dtype != dtype && y_dtype != kE4M3) return bad("Y must be of X's type or e4m3");
  if ((y_dtype == kE4M3) != (scales != nullptr) && M > 0 && N > 0)
    return bad("an e4m3 Y needs scales, and only it has them");
  if (group != 0 && group != 32 && group != 64 && group != 128)
    return bad("group must be 0 (a row), 32, 64 or 128");
  if (group != 0 && y_dtype != kE4M3) return bad("only an e4m3 Y has groups");
  // rows without columns have a scale each all the same, of 1
  if (M == 0 || (N == 0 && (!scales || group != 0))) return report_ok();
  if ((N > 0 && (!X || !Y)) || ldx < N || ldy < N || (R && ldr < N) || (H && ldh < N))
    return bad("null buffer or pitch < N");
  if (scales && ld_scales < (group ? (N + group - 1) / group : 1))
    return bad("pitch of scales < number of groups");
  if (misplaced(X, dtype) || misplaced(R, dtype) || misplaced(H, dtype) || misplaced(Y, y_dtype) ||
      (w && misplaced(w, w_dtype)) || misplaced(scales, kF32))
    return bad("buffer not aligned to its element type");
  RmsNormArgs p;
  p.X = X;
  p.R = R;
  p.w = w;
  p.H = H;
  p.Y = Y;
  p.scales = scales;
  p.ldx = ldx;
  p.ldr = ldr;
  p.ldh = ldh;
  p.ldy = ldy;
  p.lds = ld_scales;
  p.M = M;
  p.N = N;
  p.eps = eps;
  p.w_f32 = w && w_dtype == kF32;
  p.group = group;
  p.group_shift = group == 32 ? 5 : group == 64 ? 6 : 7;
  return done(rms_norm(p, dtype, static_cast<cudaStream_t>(stream)), "rms_norm");
}

int64_t b200_w4_bytes(int64_t K, int64_t N, int group, int s_dtype, int has_zeros) {
  if (const char* e = w4_shape_error(K, N, group, s_dtype)) {
    bad(e);
    return -1;
  }
  report_ok();
  return w4_layout(K, N, group, s_dtype, has_zeros).bytes();
}

int b200_w4_quantize(const float* W, int64_t ldw, int64_t K, int64_t N, int group, uint8_t* codes,
                     int64_t ldc, void* scales, int64_t lds, int s_dtype, void* stream) {
  if (const char* e = w4_shape_error(K, N, group, s_dtype)) return bad(e);
  if (K == 0 || N == 0) return report_ok();
  if (!W || !codes || !scales || ldw < N || ldc < N || lds < N)
    return bad("null buffer or pitch < N");
  if (misplaced(W, kF32) || misplaced(scales, s_dtype))
    return bad("buffer not aligned to its element type");
  return done(w4_quantize(W, ldw, K, N, group, codes, ldc, scales, lds, s_dtype,
                          static_cast<cudaStream_t>(stream)),
              "w4_quantize");
}

int b200_w4_pack(const uint8_t* codes, int64_t ldc, const void* scales, int64_t lds, int s_dtype,
                 const uint8_t* zeros, int64_t ldz, int64_t K, int64_t N, int group, void* packed,
                 void* stream) {
  if (const char* e = w4_shape_error(K, N, group, s_dtype)) return bad(e);
  if (K == 0 || N == 0) return report_ok();
  if (!codes || !scales || !packed || ldc < N || lds < N || (zeros && ldz < N))
    return bad("null buffer or pitch < N");
  if (misplaced(scales, s_dtype)) return bad("buffer not aligned to its element type");
  if (unaligned16(packed)) return bad("packed weights must be 16-byte aligned");
  // the device's context is made here, so that b200_dense_w4 can be captured
  int* status = nullptr;
  if (const int rc = device_status_word(&status)) return rc;
  return done(w4_pack(codes, ldc, scales, lds, zeros, ldz,
                      w4_layout(K, N, group, s_dtype, zeros != nullptr), packed,
                      static_cast<cudaStream_t>(stream)),
              "w4_pack");
}

int b200_w4_dequantize(const void* packed, int s_dtype, int has_zeros, int64_t K, int64_t N,
                       int group, float* W, int64_t ldw, void* stream) {
  if (const char* e = w4_shape_error(K, N, group, s_dtype)) return bad(e);
  if (K == 0 || N == 0) return report_ok();
  if (!packed || !W || ldw < N) return bad("null buffer or pitch < N");
  if (unaligned16(packed)) return bad("packed weights must be 16-byte aligned");
  if (misplaced(W, kF32)) return bad("buffer not aligned to its element type");
  return done(w4_dequantize(packed, w4_layout(K, N, group, s_dtype, has_zeros), W, ldw,
                            static_cast<cudaStream_t>(stream)),
              "w4_dequantize");
}

int b200_dense_w4(const void* X, int64_t ldx, int x_dtype, const float* x_scales,
                  int64_t ld_x_scales, int x_group, const void* packed, int s_dtype, int has_zeros,
                  int group, const void* b, int b_dtype, void* Y, int64_t ldy, int y_dtype,
                  int64_t M, int64_t N, int64_t K, int act, float alpha, void* stream) {
  if (M < 0) return bad("negative dimension");
  if (const char* e = w4_shape_error(K, N, group, s_dtype)) return bad(e);
  if (act < 0 || act > 2) return bad("unknown activation");
  if (!plain_type(x_dtype) && x_dtype != kE4M3) return bad("X must be f32, bf16, f16 or e4m3");
  if (!plain_type(y_dtype)) return bad("Y must be f32, bf16 or f16");
  if (b && !plain_type(b_dtype)) return bad("b must be f32, bf16 or f16");
  if (x_scales && x_dtype != kE4M3) return bad("only an e4m3 X has scales");
  if (x_group != 0 && x_group != 32 && x_group != 64 && x_group != 128)
    return bad("x_group must be 0 (a row), 32, 64 or 128");
  if (x_group != 0 && !x_scales) return bad("x_group without x_scales");
  if (M == 0 || N == 0) return report_ok();
  if (!Y || ldy < N) return bad("null buffer or pitch < N");
  if (K > 0 && (!X || !packed || ldx < K)) return bad("null buffer or pitch < K");
  if (x_scales && ld_x_scales < (x_group ? (K + x_group - 1) / x_group : 1))
    return bad("pitch of x_scales < number of groups");
  if (unaligned16(packed)) return bad("packed weights must be 16-byte aligned");
  if (misplaced(X, x_dtype) || misplaced(Y, y_dtype) || (b && misplaced(b, b_dtype)) ||
      misplaced(x_scales, kF32))
    return bad("buffer not aligned to its element type");
  DenseW4Args p;
  p.X = X;
  p.x_scales = x_scales;
  p.packed = packed;
  p.b = b;
  p.Y = Y;
  p.ldx = ldx;
  p.ldxs = ld_x_scales;
  p.ldy = ldy;
  p.M = M;
  p.w = w4_layout(K, N, group, s_dtype, has_zeros);
  p.x_dtype = x_dtype;
  p.x_group = x_group;
  p.b_dtype = b_dtype;
  p.y_dtype = y_dtype;
  p.act = act;
  p.alpha = alpha;
  int* status = nullptr;
  if (const int rc = device_status_word(&status)) return rc;
  return done(dense_w4(p, status, static_cast<cudaStream_t>(stream)), "dense_w4");
}

int b200_debug_w4_expire(int64_t limit_ns) {
  if (limit_ns < 0) return bad("limit_ns must not be negative");
  w4_expire(limit_ns);
  return report_ok();
}

int b200_token_logprobs(const void* logits, int64_t ld, int dtype, int64_t T, int64_t V,
                        const int32_t* tokens, float* logprobs, float* entropy, int top,
                        float* top_logprobs, int32_t* top_tokens, void* stream) {
  if (T < 0 || V < 0) return bad("negative dimension");
  if (!plain_type(dtype)) return bad("logits must be f32, bf16 or f16");
  if (top < 0 || top > kMaxTop) return bad("top must be 0 to 32");
  if ((tokens == nullptr) != (logprobs == nullptr)) return bad("logprobs go with tokens");
  if (T == 0) return report_ok();
  if (V == 0) return bad("rows without logits have no probabilities");
  if (T >= kMaxIndex / 8 || V > kMaxIndex - 64)
    return report_error(kErrTooLarge, "dimension exceeds the supported range");
  if (top > V) return bad("top exceeds the number of logits");
  if (top > 0 && (!top_logprobs || !top_tokens)) return bad("null buffer");
  if (!logits || ld < V) return bad("null buffer or pitch < V");
  if (misplaced(logits, dtype)) return bad("buffer not aligned to its element type");
  TokenLogprobsArgs p;
  p.logits = logits;
  p.ld = ld;
  p.T = T;
  p.V = V;
  p.tokens = tokens;
  p.logprobs = logprobs;
  p.entropy = entropy;
  p.top_logprobs = top_logprobs;
  p.top_tokens = top_tokens;
  p.top = top;
  return done(token_logprobs(p, dtype, static_cast<cudaStream_t>(stream)), "token_logprobs");
}

}  // extern "C"
