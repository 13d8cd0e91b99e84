// capi.cpp -- the extern "C" boundary declared in include/tsa.h.
//
// Validation happens here, before any HIP call, so argument errors are reported the same
// way on machines without a GPU.  The launch functions in kernels.h assume valid input.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "../../include/tsa.h"
#include "kernels.h"

namespace {

inline int from_hip(hipError_t e) { return e == hipSuccess ? TSA_OK : TSA_ERR_LAUNCH; }

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

// a * b * c fits in an int (workgroup counts and per-dimension products).
inline bool fits_int(long long a, long long b, long long c = 1) {
    return a >= 0 && b >= 0 && c >= 0 && a * b <= INT_MAX && a * b * c <= INT_MAX;
}

int check_attn(const void* q, const void* k, const void* v, const void* o, int B, int H, int S,
               int D, float scale, int causal, int Hkv = -1) {
    if (!q || !k || !v || !o) return TSA_ERR_NULL;
    if (Hkv == -1) Hkv = H;
    if (B < 1 || H < 1 || Hkv < 1 || S < 1 || D < 1) return TSA_ERR_SHAPE;
    if (H % Hkv != 0) return TSA_ERR_SHAPE;
    if (D != 64 && D != 128 && D != 256) return TSA_ERR_UNSUPPORTED;
    if (causal != 0 && causal != 1) return TSA_ERR_ARG;
    // The running max is taken over raw q.k, which is the max of the scaled scores only
    // for scale > 0 (the reference's scale is 1/sqrt(D), src/attn_sm75.cu:462).
    if (!(scale > 0.f) || !std::isfinite(scale)) return TSA_ERR_ARG;
    // workgroups: B*H*ceil(S/128) for the MFMA kernel, B*H*ceil(S/64) for the VALU one,
    // B*H*S/128 for the naive one
    if (!fits_int(B, H, S)) return TSA_ERR_SHAPE;
    return TSA_OK;
}

int check_gdn(const void* q, const void* k, const void* v, const float* g, const float* beta,
              const float* state, const void* out, int B, int T, int Hq, int Hv, int dk, int dv,
              float scale) {
    if (!q || !k || !v || !g || !beta || !state || !out) return TSA_ERR_NULL;
    if (B < 1 || T < 1 || Hq < 1 || Hv < 1 || dk < 1 || dv < 1) return TSA_ERR_SHAPE;
    if (!std::isfinite(scale)) return TSA_ERR_ARG;
    // element offsets are 64-bit in every kernel; only workgroup counts must fit an int
    if (!fits_int(B, Hv, dv)) return TSA_ERR_SHAPE;
    return TSA_OK;
}

// The raw gate inputs of the fused pre-ops and the l2-norm eps.
int check_gates(const float* a, const float* b, const float* dt_bias, const float* A, float eps) {
    if (!a || !b || !dt_bias || !A) return TSA_ERR_NULL;
    if (!(eps > 0.f) || !std::isfinite(eps)) return TSA_ERR_ARG;
    return TSA_OK;
}

}  // namespace

extern "C" const char* tsa_strerror(int code) {
    switch (code) {
        case TSA_OK: return "ok";
        case TSA_ERR_NULL: return "a required pointer is NULL";
        case TSA_ERR_SHAPE: return "invalid shape (size < 1, too large, or inconsistent)";
        case TSA_ERR_UNSUPPORTED: return "shape not supported by this library (attention: D in {64,128,256}; GDN: dk = dv = 128, chunk = 64)";
        case TSA_ERR_WORKSPACE: return "workspace is NULL or smaller than the required size";
        case TSA_ERR_LAUNCH: return "the HIP runtime rejected a kernel launch";
        case TSA_ERR_ARG: return "invalid argument (causal not 0/1, scale not finite / not > 0, eps not finite / not > 0, rows or 8-bit cache: a misaligned buffer or stride, top < first + recent + 1, rotary positions: a parameter out of its range)";
        case TSA_ERR_SCRATCH: return "the shapes need more than the 64 MiB device scratch of tsa_gdn_chunked_fwd_noalloc (use tsa_gdn_chunked_fwd with a workspace)";
        default: return "unknown tsa error code";
    }
}

extern "C" const char* tsa_version(void) { return "tsa 0.1 gfx950"; }

extern "C" int tsa_attn_fwd(const void* q, const void* k, const void* v, void* o, int B, int H,
                            int S, int D, float scale, int causal, void* stream) {
    const int rc = check_attn(q, k, v, o, B, H, S, D, scale, causal);
    if (rc) return rc;
    return from_hip(tsa::attn_fwd(q, k, v, nullptr, o, B, H, H, S, D, scale, causal,
                                  as_stream(stream)));
}

extern "C" int tsa_attn_naive(const void* q, const void* k, const void* v, void* o, int B,
                              int H, int S, int D, float scale, int causal, void* stream) {
    const int rc = check_attn(q, k, v, o, B, H, S, D, scale, causal);
    if (rc) return rc;
    return from_hip(tsa::attn_naive(q, k, v, nullptr, o, B, H, H, S, D, scale, causal,
                                    as_stream(stream)));
}

extern "C" int tsa_attn_fwd_valu(const void* q, const void* k, const void* v, void* o, int B,
                                 int H, int S, int D, float scale, int causal, void* stream) {
    const int rc = check_attn(q, k, v, o, B, H, S, D, scale, causal);
    if (rc) return rc;
    return from_hip(tsa::attn_valu(q, k, v, o, B, H, S, D, scale, causal, as_stream(stream)));
}

extern "C" int tsa_attn_gqa_fwd(const void* q, const void* k, const void* v, const void* gate,
                                void* o, int B, int Hq, int Hkv, int S, int D, float scale,
                                int causal, void* stream) {
    const int rc = check_attn(q, k, v, o, B, Hq, S, D, scale, causal, Hkv);
    if (rc) return rc;
    return from_hip(tsa::attn_fwd(q, k, v, gate, o, B, Hq, Hkv, S, D, scale, causal,
                                  as_stream(stream)));
}

extern "C" int tsa_attn_gqa_naive(const void* q, const void* k, const void* v, const void* gate,
                                  void* o, int B, int Hq, int Hkv, int S, int D, float scale,
                                  int causal, void* stream) {
    const int rc = check_attn(q, k, v, o, B, Hq, S, D, scale, causal, Hkv);
    if (rc) return rc;
    return from_hip(tsa::attn_naive(q, k, v, gate, o, B, Hq, Hkv, S, D, scale, causal,
                                    as_stream(stream)));
}

extern "C" size_t tsa_gdn_chunked_workspace_bytes(int B, int T, int Hq, int Hv, int dk, int dv,
                                                  int chunk) {
    if (B < 1 || T < 1 || Hq < 1 || Hv < 1 || dk != 128 || dv != 128 || chunk != 64) return 0;
    return tsa::gdn_chunked_ws_bytes(B, T, Hv, false);
}

extern "C" size_t tsa_gdn_chunked_workspace_bytes_f32(int B, int T, int Hq, int Hv, int dk, int dv,
                                                      int chunk) {
    if (B < 1 || T < 1 || Hq < 1 || Hv < 1 || dk != 128 || dv != 128 || chunk != 64) return 0;
    return tsa::gdn_chunked_ws_bytes(B, T, Hv, true);
}

extern "C" size_t tsa_gdn_chunked_plan_workspace_bytes(int B, int T, int Hq, int Hv, int dk, int dv,
                                                       int chunk, int io_f32, int nseg) {
    if (B < 1 || T < 1 || Hq < 1 || Hv < 1 || dk != 128 || dv != 128 || chunk != 64) return 0;
    if ((io_f32 != 0 && io_f32 != 1) || nseg < 0) return 0;
    return tsa::gdn_chunked_ws_bytes(B, T, Hv, io_f32 != 0, nseg);
}

namespace {
int chunked(const void* q, const void* k, const void* v, const float* g_log, const float* beta,
            float* state, void* out, int B, int T, int Hq, int Hv, int dk, int dv, int chunk,
            float scale, void* ws, size_t ws_bytes, bool f32, void* stream, int nseg = 0) {
    int rc = check_gdn(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, scale);
    if (rc) return rc;
    if (chunk < 1) return TSA_ERR_SHAPE;
    if (dk != 128 || dv != 128 || chunk != 64) return TSA_ERR_UNSUPPORTED;
    if (nseg < 0) return TSA_ERR_ARG;
    const long long nch = (T + 63LL) / 64;
    if (!fits_int(B, Hv, nch) || !fits_int(B, Hv, 8)) return TSA_ERR_SHAPE;
    const size_t need = tsa::gdn_chunked_ws_bytes(B, T, Hv, f32, nseg);
    if (!ws || ws_bytes < need) return TSA_ERR_WORKSPACE;
    return from_hip(tsa::gdn_chunked(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, scale, ws, f32,
                                     as_stream(stream), nseg));
}
}  // namespace

extern "C" int tsa_gdn_chunked_plan_fwd(const void* q, const void* k, const void* v,
                                        const float* g_log, const float* beta, float* state, void* out,
                                        int B, int T, int Hq, int Hv, int dk, int dv, int chunk,
                                        float scale, int io_f32, int nseg, void* ws, size_t ws_bytes,
                                        void* stream) {
    if (io_f32 != 0 && io_f32 != 1) return TSA_ERR_ARG;
    return chunked(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, chunk, scale, ws, ws_bytes,
                   io_f32 != 0, stream, nseg);
}

extern "C" int tsa_gdn_chunked_fwd(const void* q, const void* k, const void* v,
                                   const float* g_log, const float* beta, float* state, void* out,
                                   int B, int T, int Hq, int Hv, int dk, int dv, int chunk,
                                   float scale, void* ws, size_t ws_bytes, void* stream) {
    return chunked(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, chunk, scale, ws, ws_bytes,
                   false, stream);
}

extern "C" int tsa_gdn_chunked_fwd_f32(const float* q, const float* k, const float* v,
                                       const float* g_log, const float* beta, float* state, float* out,
                                       int B, int T, int Hq, int Hv, int dk, int dv, int chunk,
                                       float scale, void* ws, size_t ws_bytes, void* stream) {
    return chunked(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, chunk, scale, ws, ws_bytes,
                   true, stream);
}

extern "C" int tsa_gdn_chunked_fwd_noalloc(const void* q, const void* k, const void* v,
                                           const float* g_log, const float* beta, float* state,
                                           void* out, int B, int T, int Hq, int Hv, int dk, int dv,
                                           int chunk, float scale, void* stream) {
    int rc = check_gdn(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, scale);
    if (rc) return rc;
    if (chunk < 1) return TSA_ERR_SHAPE;
    if (dk != 128 || dv != 128 || chunk != 64) return TSA_ERR_UNSUPPORTED;
    const long long nch = (T + 63LL) / 64;
    if (!fits_int(B, Hv, nch) || !fits_int(B, Hv, 8)) return TSA_ERR_SHAPE;
    if (tsa::gdn_chunked_noalloc_ws_bytes(B, T, Hv) > tsa::gdn_chunked_noalloc_max_bytes()) return TSA_ERR_SCRATCH;
    return from_hip(tsa::gdn_chunked_noalloc(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, scale,
                                             as_stream(stream)));
}

extern "C" int tsa_gdn_chunked_redo_count(const void* ws, size_t ws_bytes, int B, int T, int Hq,
                                          int Hv, int dk, int dv, int chunk, int io_f32, int* count,
                                          void* stream) {
    if (!ws || !count) return TSA_ERR_NULL;
    if (B < 1 || T < 1 || Hq < 1 || Hv < 1 || chunk < 1) return TSA_ERR_SHAPE;
    if (dk != 128 || dv != 128 || chunk != 64) return TSA_ERR_UNSUPPORTED;
    if (io_f32 != 0 && io_f32 != 1) return TSA_ERR_ARG;
    const long long nch = (T + 63LL) / 64;
    if (!fits_int(B, Hv, nch) || !fits_int(B, Hv, 8)) return TSA_ERR_SHAPE;
    if (ws_bytes < tsa::gdn_chunked_ws_bytes(B, T, Hv, io_f32 != 0)) return TSA_ERR_WORKSPACE;
    return from_hip(tsa::gdn_chunked_redo_count(ws, B, T, Hv, io_f32 != 0, count, as_stream(stream)));
}

namespace {
int recurrent(const void* q, const void* k, const void* v, const float* g_log, const float* beta,
              float* state, void* out, int B, int T, int Hq, int Hv, int dk, int dv, float scale,
              bool f32, void* stream) {
    int rc = check_gdn(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, scale);
    if (rc) return rc;
    if (dk != 128 || dv != 128) return TSA_ERR_UNSUPPORTED;
    if (!fits_int(B, Hv, 4)) return TSA_ERR_SHAPE;
    return from_hip(tsa::gdn_recurrent(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, scale, f32,
                                       as_stream(stream)));
}

int naive(const void* q, const void* k, const void* v, const float* g_log, const float* beta,
          float* state, void* out, int B, int T, int Hq, int Hv, int dk, int dv, float scale,
          bool f32, void* stream) {
    int rc = check_gdn(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, scale);
    if (rc) return rc;
    return from_hip(tsa::gdn_naive(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, scale, f32,
                                   as_stream(stream)));
}
}  // namespace

extern "C" int tsa_gdn_recurrent_fwd(const void* q, const void* k, const void* v,
                                     const float* g_log, const float* beta, float* state,
                                     void* out, int B, int T, int Hq, int Hv, int dk, int dv,
                                     float scale, void* stream) {
    return recurrent(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, scale, false, stream);
}

extern "C" int tsa_gdn_recurrent_fwd_f32(const float* q, const float* k, const float* v,
                                         const float* g_log, const float* beta, float* state,
                                         float* out, int B, int T, int Hq, int Hv, int dk, int dv,
                                         float scale, void* stream) {
    return recurrent(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, scale, true, stream);
}

extern "C" int tsa_gdn_decode_step(const void* q, const void* k, const void* v,
                                   const float* g_log, const float* beta, float* state, void* out,
                                   int B, int Hq, int Hv, int dk, int dv, float scale,
                                   void* stream) {
    return recurrent(q, k, v, g_log, beta, state, out, B, 1, Hq, Hv, dk, dv, scale, false, stream);
}

extern "C" int tsa_gdn_decode_step_f32(const float* q, const float* k, const float* v,
                                       const float* g_log, const float* beta, float* state,
                                       float* out, int B, int Hq, int Hv, int dk, int dv, float scale,
                                       void* stream) {
    return recurrent(q, k, v, g_log, beta, state, out, B, 1, Hq, Hv, dk, dv, scale, true, stream);
}

extern "C" int tsa_gdn_naive(const void* q, const void* k, const void* v, const float* g_log,
                             const float* beta, float* state, void* out, int B, int T, int Hq,
                             int Hv, int dk, int dv, float scale, void* stream) {
    return naive(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, scale, false, stream);
}

extern "C" int tsa_gdn_naive_f32(const float* q, const float* k, const float* v, const float* g_log,
                                 const float* beta, float* state, float* out, int B, int T, int Hq,
                                 int Hv, int dk, int dv, float scale, void* stream) {
    return naive(q, k, v, g_log, beta, state, out, B, T, Hq, Hv, dk, dv, scale, true, stream);
}

extern "C" int tsa_gdn_chunked_fused_fwd(const void* q, const void* k, const void* v, const float* a,
                                         const float* b, const float* dt_bias, const float* A,
                                         float* state, void* out, int B, int T, int Hq, int Hv,
                                         int dk, int dv, int chunk, float scale, float eps, void* ws,
                                         size_t ws_bytes, void* stream) {
    int rc = check_gdn(q, k, v, a, b, state, out, B, T, Hq, Hv, dk, dv, scale);
    if (rc) return rc;
    rc = check_gates(a, b, dt_bias, A, eps);
    if (rc) return rc;
    if (chunk < 1) return TSA_ERR_SHAPE;
    if (dk != 128 || dv != 128 || chunk != 64) return TSA_ERR_UNSUPPORTED;
    const long long nch = (T + 63LL) / 64;
    if (!fits_int(B, Hv, nch) || !fits_int(B, Hv, 8)) return TSA_ERR_SHAPE;
    const size_t need = tsa::gdn_chunked_ws_bytes(B, T, Hv, false);
    if (!ws || ws_bytes < need) return TSA_ERR_WORKSPACE;
    return from_hip(tsa::gdn_chunked_fused(q, k, v, tsa::GdnRawGates{a, b, dt_bias, A, eps}, state,
                                           out, B, T, Hq, Hv, scale, ws, as_stream(stream)));
}

extern "C" int tsa_gdn_decode_fused_step(const void* q, const void* k, const void* v, const float* a,
                                         const float* b, const float* dt_bias, const float* A,
                                         float* state, void* out, int B, int Hq, int Hv, int dk,
                                         int dv, float scale, float eps, void* stream) {
    int rc = check_gdn(q, k, v, a, b, state, out, B, 1, Hq, Hv, dk, dv, scale);
    if (rc) return rc;
    rc = check_gates(a, b, dt_bias, A, eps);
    if (rc) return rc;
    if (dk != 128 || dv != 128) return TSA_ERR_UNSUPPORTED;
    if (!fits_int(B, Hv, 8)) return TSA_ERR_SHAPE;
    return from_hip(tsa::gdn_decode_fused(q, k, v, tsa::GdnRawGates{a, b, dt_bias, A, eps}, state,
                                          out, B, Hq, Hv, scale, as_stream(stream)));
}

extern "C" int tsa_gdn_preprocess(const void* q, const void* k, const float* a, const float* b,
                                  const float* dt_bias, const float* A, void* q_out, void* k_out,
                                  float* g_log, float* beta, int B, int T, int Hq, int Hv, int dk,
                                  float eps, void* stream) {
    if (!q || !k || !q_out || !k_out || !g_log || !beta) return TSA_ERR_NULL;
    int rc = check_gates(a, b, dt_bias, A, eps);
    if (rc) return rc;
    if (B < 1 || T < 1 || Hq < 1 || Hv < 1 || dk < 1) return TSA_ERR_SHAPE;
    if (dk != 128) return TSA_ERR_UNSUPPORTED;
    // workgroups: 2 * B*T*Hq / 16 rows and B*T*Hv / 256 gates
    if (!fits_int(B, T, Hq) || !fits_int(B, T, Hv)) return TSA_ERR_SHAPE;
    return from_hip(tsa::gdn_preprocess(q, k, a, b, dt_bias, A, q_out, k_out, g_log, beta, B, T, Hq,
                                        Hv, eps, as_stream(stream)));
}

extern "C" int tsa_gdn_gated_rmsnorm(const void* x, const void* z, const float* w, void* y, int B,
                                     int T, int Hv, int dv, float eps, void* stream) {
    if (!x || !z || !w || !y) return TSA_ERR_NULL;
    if (B < 1 || T < 1 || Hv < 1 || dv < 1) return TSA_ERR_SHAPE;
    if (dv != 128) return TSA_ERR_UNSUPPORTED;
    if (!(eps > 0.f) || !std::isfinite(eps)) return TSA_ERR_ARG;
    if (!fits_int(B, T, Hv)) return TSA_ERR_SHAPE;
    return from_hip(tsa::gdn_gated_rmsnorm(x, z, w, y, B, T, Hv, eps, as_stream(stream)));
}

// ---- the 8-bit K/V cache ----
namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_kv8(const tsa_kv8* c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_sum || !c->k_sum_scale || !c->k_open || !c->v_open || !c->table)
        return TSA_ERR_NULL;
    if (c->B < 1 || c->Hkv < 1 || c->D < 1 || c->n_pages < 1 || c->max_blocks < 1) return TSA_ERR_SHAPE;
    if (c->D != 64 && c->D != 128 && c->D != 256) return TSA_ERR_UNSUPPORTED;
    // positions are ints, a workgroup per (sequence, K or V, head) at least
    if (c->max_blocks > INT_MAX / 64 - 1 || !fits_int(c->B, c->Hkv) || c->B > 65535 || c->Hkv > 32767 ||
        (long long)c->B * c->Hkv > 65535)
        return TSA_ERR_SHAPE;
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_sum) || !aligned16(c->k_open) || !aligned16(c->v_open))
        return TSA_ERR_ARG;
    return TSA_OK;
}

int check_rows(const tsa_rows* r, int B, int H, int T, bool out) {
    if (!r || !r->data) return TSA_ERR_NULL;
    if (!aligned16(r->data)) return TSA_ERR_ARG;
    const int64_t stride[3] = {r->stride_b, r->stride_h, r->stride_t};
    const int size[3] = {B, H, T};
    for (int i = 0; i < 3; ++i)
        if (size[i] > 1 && (stride[i] < (out ? 1 : 0) || stride[i] % 8 != 0)) return TSA_ERR_ARG;
    return TSA_OK;
}

tsa::Kv8 as_kv8(const tsa_kv8* c) {
    return {static_cast<unsigned char*>(c->k), static_cast<unsigned char*>(c->v), c->k_scale, c->v_scale,
            static_cast<signed char*>(c->k_sum), c->k_sum_scale, static_cast<_Float16*>(c->k_open),
            static_cast<_Float16*>(c->v_open), c->table, c->B, c->Hkv, c->D, c->n_pages, c->max_blocks};
}

// Strides of dimensions of one row are not looked at by the caller: 0 here, so that none is used.
tsa::Rows16 as_rows(const tsa_rows* r, int B, int H, int T) {
    if (!r || !r->data) return {nullptr, 0, 0, 0};
    return {static_cast<_Float16*>(r->data), B > 1 ? r->stride_b : 0, H > 1 ? r->stride_h : 0, T > 1 ? r->stride_t : 0};
}

// Queries: rows of all heads must fit an int, and a group's elements too.
int check_kv8_queries(const tsa_kv8* c, int T, int Hq) {
    if (T < 1 || Hq < 1 || Hq % c->Hkv != 0 || Hq / c->Hkv > 65536) return TSA_ERR_SHAPE;
    return fits_int(c->B, Hq, T) ? TSA_OK : TSA_ERR_SHAPE;
}

// Entries of a list: the kernels count parts of blocks in ints.
bool fits_top(int top) { return top >= 1 && top <= 1 << 24; }

int check_ws(const void* ws, size_t ws_bytes, size_t need) {
    if (need && (!ws || ws_bytes < need)) return TSA_ERR_WORKSPACE;
    return need && !aligned16(ws) ? TSA_ERR_ARG : TSA_OK;
}

int kv8_nb(const tsa_kv8* c, int max_len) {
    const int nb = (int)((max_len + 63LL) / 64);
    return nb < c->max_blocks ? nb : c->max_blocks;
}

int check_kv8_attn(const tsa_kv8* c, const tsa_rows* q, const tsa_rows* gate, const tsa_rows* o, const int32_t* len,
                   int T, int Hq, float scale) {
    int rc = check_kv8(c);
    if (rc) return rc;
    if (!len) return TSA_ERR_NULL;
    if ((rc = check_kv8_queries(c, T, Hq))) return rc;
    if ((rc = check_rows(q, c->B, Hq, T, false)) || (rc = check_rows(o, c->B, Hq, T, true))) return rc;
    if (gate && (rc = check_rows(gate, c->B, Hq, T, false))) return rc;
    if (!(scale > 0.f) || !std::isfinite(scale)) return TSA_ERR_ARG;
    return TSA_OK;
}

}  // namespace

extern "C" int tsa_kv8_write(const tsa_kv8* cache, const tsa_rows* k, const tsa_rows* v, const int32_t* len,
                             const int32_t* n_new, int T, void* stream) {
    int rc = check_kv8(cache);
    if (rc) return rc;
    if (!len) return TSA_ERR_NULL;
    if (T < 1 || T > INT_MAX - 64) return TSA_ERR_SHAPE;
    if ((rc = check_rows(k, cache->B, cache->Hkv, T, false)) || (rc = check_rows(v, cache->B, cache->Hkv, T, false))) return rc;
    return from_hip(tsa::kv8_write(as_kv8(cache), as_rows(k, cache->B, cache->Hkv, T), as_rows(v, cache->B, cache->Hkv, T),
                                   len, n_new, T, as_stream(stream)));
}

extern "C" int tsa_kv8_read(const tsa_kv8* cache, const int32_t* len, const int32_t* start, int S, const tsa_rows* k,
                            const tsa_rows* v, void* stream) {
    int rc = check_kv8(cache);
    if (rc) return rc;
    if (!len || (!k && !v)) return TSA_ERR_NULL;
    if (S < 1 || S > INT_MAX - 64) return TSA_ERR_SHAPE;
    if (k && (rc = check_rows(k, cache->B, cache->Hkv, S, true))) return rc;
    if (v && (rc = check_rows(v, cache->B, cache->Hkv, S, true))) return rc;
    return from_hip(tsa::kv8_read(as_kv8(cache), len, start, S, as_rows(k, cache->B, cache->Hkv, S),
                                  as_rows(v, cache->B, cache->Hkv, S), as_stream(stream)));
}

extern "C" size_t tsa_kv8_workspace_bytes(const tsa_kv8* cache, int T, int Hq, int max_len, int top) {
    if (check_kv8(cache) || check_kv8_queries(cache, T, Hq) || max_len < 1 || (top != 0 && !fits_top(top))) return 0;
    const int nb = kv8_nb(cache, max_len);
    return top != 0 && !fits_int(T, nb) ? 0 : tsa::kv8_ws_bytes(as_kv8(cache), T, Hq, nb, top);
}

extern "C" int tsa_attn_kv8_fwd(const tsa_kv8* cache, const tsa_rows* q, const tsa_rows* gate, const tsa_rows* o,
                                const int32_t* len, const int32_t* n_new, int T, int Hq, int max_len, float scale,
                                int causal, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_kv8_attn(cache, q, gate, o, len, T, Hq, scale);
    if (rc) return rc;
    if (max_len < 1) return TSA_ERR_SHAPE;
    if (causal != 0 && causal != 1) return TSA_ERR_ARG;
    const int B = cache->B, nb = kv8_nb(cache, max_len);
    const size_t need = tsa::kv8_ws_bytes(as_kv8(cache), T, Hq, nb, 0);
    if ((rc = check_ws(ws, ws_bytes, need))) return rc;
    return from_hip(tsa::kv8_attn(as_kv8(cache), as_rows(q, B, Hq, T), as_rows(gate, B, Hq, T), as_rows(o, B, Hq, T), len,
                                  n_new, T, Hq, nb, scale, causal, ws, as_stream(stream)));
}

extern "C" int tsa_kv8_select(const tsa_kv8* cache, const tsa_rows* q, const int32_t* len, const int32_t* n_new, int T,
                              int Hq, int top, int first, int recent, int32_t* blocks, int max_len, void* ws,
                              size_t ws_bytes, void* stream) {
    int rc = check_kv8(cache);
    if (rc) return rc;
    if (!len || !blocks) return TSA_ERR_NULL;
    if ((rc = check_kv8_queries(cache, T, Hq))) return rc;
    if (max_len < 1 || !fits_top(top) || first < 0 || recent < 0) return TSA_ERR_SHAPE;
    if ((long long)first + recent + 1 > top) return TSA_ERR_ARG;
    const int B = cache->B, nb = kv8_nb(cache, max_len);
    if (!fits_int(T, nb)) return TSA_ERR_SHAPE;  // a query's scores of all blocks: the launch's workgroups
    if ((rc = check_rows(q, B, Hq, T, false))) return rc;
    const size_t need = tsa::kv8_ws_bytes(as_kv8(cache), T, Hq, nb, top);
    if ((rc = check_ws(ws, ws_bytes, need))) return rc;
    return from_hip(tsa::kv8_select(as_kv8(cache), as_rows(q, B, Hq, T), len, n_new, T, Hq, top, first, recent, blocks, nb,
                                    ws, as_stream(stream)));
}

extern "C" int tsa_attn_kv8_blocks_fwd(const tsa_kv8* cache, const tsa_rows* q, const tsa_rows* gate, const tsa_rows* o,
                                       const int32_t* len, const int32_t* n_new, int T, int Hq, const int32_t* blocks,
                                       int top, float scale, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_kv8_attn(cache, q, gate, o, len, T, Hq, scale);
    if (rc) return rc;
    if (!blocks) return TSA_ERR_NULL;
    if (!fits_top(top)) return TSA_ERR_SHAPE;
    const int B = cache->B;
    const size_t need = tsa::kv8_ws_bytes(as_kv8(cache), T, Hq, 1, top);
    if ((rc = check_ws(ws, ws_bytes, need))) return rc;
    return from_hip(tsa::kv8_attn_blocks(as_kv8(cache), as_rows(q, B, Hq, T), as_rows(gate, B, Hq, T), as_rows(o, B, Hq, T),
                                         len, n_new, T, Hq, blocks, top, scale, ws, as_stream(stream)));
}

// ---- rotary positions ----
extern "C" int tsa_rope_freqs(const tsa_rope_params* p, uint64_t* freq, float* amp) {
    if (!p || !freq || !amp) return TSA_ERR_NULL;
    if (p->rot < 2 || p->rot % 2 != 0) return TSA_ERR_SHAPE;
    if (!(p->base > 1.0) || !std::isfinite(p->base)) return TSA_ERR_ARG;
    const int kind = p->scaling;
    if (kind < TSA_ROPE_PLAIN || kind > TSA_ROPE_WAVELENGTH) return TSA_ERR_ARG;
    if (kind != TSA_ROPE_PLAIN && (!(p->factor >= 1.0) || !std::isfinite(p->factor))) return TSA_ERR_ARG;
    if (kind == TSA_ROPE_NTK && p->rot < 4) return TSA_ERR_ARG;
    if ((kind == TSA_ROPE_YARN || kind == TSA_ROPE_WAVELENGTH) && p->orig_len < 1) return TSA_ERR_ARG;
    if (kind == TSA_ROPE_YARN && !(p->beta_slow > 0.0 && p->beta_fast > p->beta_slow && std::isfinite(p->beta_fast))) return TSA_ERR_ARG;
    if (kind == TSA_ROPE_WAVELENGTH && !(p->low > 0.0 && p->high > p->low && std::isfinite(p->high))) return TSA_ERR_ARG;
    // in the host's widest floats (64 bits of mantissa): the result has as many
    const long double pi = 3.14159265358979323846264338327950288L;
    const long double R = p->rot, s = p->factor, n = p->orig_len;
    const long double base = kind == TSA_ROPE_NTK ? p->base * std::pow(s, R / (R - 2)) : (long double)p->base;
    long double lo = 0, hi = 0;
    if (kind == TSA_ROPE_YARN) {
        auto pair_that_turns = [&](long double times) { return R * std::log(n / (times * 2 * pi)) / (2 * std::log(base)); };
        lo = std::max(std::floor(pair_that_turns(p->beta_fast)), 0.0L);
        hi = std::min(std::ceil(pair_that_turns(p->beta_slow)), R - 1);
    }
    for (int i = 0; i < p->rot / 2; ++i) {
        long double f = std::pow(base, -2.0L * i / R);
        if (kind == TSA_ROPE_LINEAR) f /= s;
        if (kind == TSA_ROPE_YARN) {
            const long double ramp = std::min(std::max((i - lo) / std::max(hi - lo, 0.001L), 0.0L), 1.0L);
            f = f * (1 - ramp) + f / s * ramp;
        }
        if (kind == TSA_ROPE_WAVELENGTH) {
            const long double turns = n * f / (2 * pi);
            const long double keep = std::min(std::max((turns - p->low) / ((long double)p->high - p->low), 0.0L), 1.0L);
            f = f * keep + f / s * (1 - keep);
        }
        freq[i] = (uint64_t)std::floor(f / (2 * pi) * 18446744073709551616.0L + 0.5L);  // f <= 1 radian: below 2^62
    }
    *amp = kind == TSA_ROPE_YARN ? (float)(0.1L * std::log(s) + 1) : 1.f;
    return TSA_OK;
}

namespace {

tsa::RopeRows as_rope(const tsa_rows* r, int B, int H, int T) {
    const tsa::Rows16 x = as_rows(r, B, H, T);
    return {x.data, x.b, x.h, x.t};
}

// An input and its output: apart, or the same rows.
int check_rope(const tsa_rows* x, const tsa_rows* y, int B, int H, int T) {
    int rc = check_rows(x, B, H, T, false);
    if (rc || (rc = check_rows(y, B, H, T, true))) return rc;
    if (x->data != y->data) return TSA_OK;
    const tsa::RopeRows a = as_rope(x, B, H, T), b = as_rope(y, B, H, T);
    return a.b == b.b && a.h == b.h && a.t == b.t ? TSA_OK : TSA_ERR_ARG;
}

}  // namespace

extern "C" int tsa_rope(const tsa_rope_plan* plan, int type, const tsa_rows* q, const tsa_rows* q_out, int Hq, const tsa_rows* k,
                        const tsa_rows* k_out, int Hk, const int32_t* pos, const int32_t* len, const int32_t* n_new, int B, int T,
                        int D, int back, void* stream) {
    if (!plan || !plan->freq) return TSA_ERR_NULL;
    if (B < 1 || T < 1 || Hq < 1 || Hk < 0 || D < 1) return TSA_ERR_SHAPE;
    if (D != 64 && D != 128 && D != 256) return TSA_ERR_UNSUPPORTED;
    if (plan->rot < 2 || plan->rot % 2 != 0 || plan->rot > D) return TSA_ERR_SHAPE;
    if (plan->interleaved != 0 && plan->interleaved != 1) return TSA_ERR_ARG;
    if (!std::isfinite(plan->amp) || (type != TSA_TYPE_F16 && type != TSA_TYPE_F32) || (back != 0 && back != 1)) return TSA_ERR_ARG;
    // rows of all sequences, and a workgroup's units of all heads, in ints
    if (!fits_int(B, T, D) || (long long)Hq + Hk > 65535) return TSA_ERR_SHAPE;
    int rc = check_rope(q, q_out, B, Hq, T);
    if (rc) return rc;
    if (Hk > 0 && (rc = check_rope(k, k_out, B, Hk, T))) return rc;
    const tsa::RopeRows none = {nullptr, 0, 0, 0};
    static_assert(sizeof(unsigned long long) == sizeof(uint64_t), "the table's type");
    return from_hip(tsa::rope(reinterpret_cast<const unsigned long long*>(plan->freq), plan->amp, plan->rot, plan->interleaved,
                              type == TSA_TYPE_F32, as_rope(q, B, Hq, T), as_rope(q_out, B, Hq, T), Hq,
                              Hk ? as_rope(k, B, Hk, T) : none, Hk ? as_rope(k_out, B, Hk, T) : none, Hk, pos, len, n_new, B, T, D,
                              back, as_stream(stream)));
}

// ---- attention's training pair ----
namespace {

int check_train_sizes(int B, int Hq, int Hkv, int Tq, int Tk, int D) {
    if (B < 1 || Hq < 1 || Hkv < 1 || Tq < 1 || Tk < 1 || D < 1 || Hq % Hkv != 0) return TSA_ERR_SHAPE;
    if (D != 64 && D != 128 && D != 256) return TSA_ERR_UNSUPPORTED;
    // rows of all heads, and positions, in ints; a launch's threads, up to 512 for 32 rows, below 2^32
    if (!fits_int(B, Hq, Tq) || !fits_int(B, Hkv, Tk) || (long long)Tq + Tk > INT_MAX - 1024) return TSA_ERR_SHAPE;
    return (long long)B * ((long long)Hq * ((Tq + 31) / 32) + (long long)Hkv * ((Tk + 31) / 32)) < 1 << 23 ? TSA_OK : TSA_ERR_SHAPE;
}

// Rows whose tiles are copied: offsets within a tile of 64 rows fit 32 bits.
int check_tile_rows(const tsa_rows* r, int B, int H, int T, bool out) {
    const int rc = check_rows(r, B, H, T, out);
    if (rc) return rc;
    return T > 1 && r->stride_t > 1 << 24 ? TSA_ERR_SHAPE : TSA_OK;
}

int check_train(const tsa_rows* q, const tsa_rows* k, const tsa_rows* v, const tsa_rows* gate, const tsa_rows* o, const float* lse,
                int B, int Hq, int Hkv, int Tq, int Tk, int D, float scale, int causal, bool fwd) {
    int rc = check_train_sizes(B, Hq, Hkv, Tq, Tk, D);
    if (rc) return rc;
    if (!lse) return TSA_ERR_NULL;
    if ((rc = check_tile_rows(q, B, Hq, Tq, false)) || (rc = check_tile_rows(k, B, Hkv, Tk, false)) ||
        (rc = check_tile_rows(v, B, Hkv, Tk, false)) || (rc = check_tile_rows(o, B, Hq, Tq, fwd)))
        return rc;
    if (gate && (rc = check_tile_rows(gate, B, Hq, Tq, false))) return rc;
    if ((causal != 0 && causal != 1) || !(scale > 0.f) || !std::isfinite(scale)) return TSA_ERR_ARG;
    return TSA_OK;
}

}  // namespace

extern "C" int tsa_attn_train_fwd(const tsa_rows* q, const tsa_rows* k, const tsa_rows* v, const tsa_rows* gate, const tsa_rows* o,
                                  float* lse, const int32_t* len_q, const int32_t* len_k, int B, int Hq, int Hkv, int Tq, int Tk,
                                  int D, float scale, int causal, void* stream) {
    const int rc = check_train(q, k, v, gate, o, lse, B, Hq, Hkv, Tq, Tk, D, scale, causal, true);
    if (rc) return rc;
    return from_hip(tsa::attn_train_fwd(as_rows(q, B, Hq, Tq), as_rows(k, B, Hkv, Tk), as_rows(v, B, Hkv, Tk), as_rows(gate, B, Hq, Tq),
                                        as_rows(o, B, Hq, Tq), lse, len_q, len_k, B, Hq, Hkv, Tq, Tk, D, scale, causal,
                                        as_stream(stream)));
}

extern "C" size_t tsa_attn_bwd_workspace_bytes(int B, int Hq, int Hkv, int Tq, int Tk, int D, int gated, int causal) {
    if (check_train_sizes(B, Hq, Hkv, Tq, Tk, D) || (gated != 0 && gated != 1) || (causal != 0 && causal != 1)) return 0;
    return tsa::attn_bwd_ws_bytes(B, Hq, Hkv, Tq, Tk, D, gated != 0, causal != 0);
}

extern "C" int tsa_attn_bwd(const tsa_rows* d_out, const tsa_rows* q, const tsa_rows* k, const tsa_rows* v, const tsa_rows* gate,
                            const tsa_rows* o, const float* lse, const tsa_rows* dq, const tsa_rows* dk, const tsa_rows* dv,
                            const tsa_rows* dgate, const int32_t* len_q, const int32_t* len_k, int B, int Hq, int Hkv, int Tq,
                            int Tk, int D, float scale, int causal, void* ws, size_t ws_bytes, void* stream) {
    int rc = check_train(q, k, v, gate, o, lse, B, Hq, Hkv, Tq, Tk, D, scale, causal, false);
    if (rc) return rc;
    if ((rc = check_tile_rows(d_out, B, Hq, Tq, false)) || (rc = check_tile_rows(dq, B, Hq, Tq, true)) ||
        (rc = check_tile_rows(dk, B, Hkv, Tk, true)) || (rc = check_tile_rows(dv, B, Hkv, Tk, true)))
        return rc;
    if (gate && (rc = check_tile_rows(dgate, B, Hq, Tq, true))) return rc;
    if ((rc = check_ws(ws, ws_bytes, tsa::attn_bwd_ws_bytes(B, Hq, Hkv, Tq, Tk, D, gate != nullptr, causal != 0)))) return rc;
    const tsa::AttnRows x = {as_rows(q, B, Hq, Tq), as_rows(k, B, Hkv, Tk), as_rows(v, B, Hkv, Tk), as_rows(gate, B, Hq, Tq),
                             as_rows(o, B, Hq, Tq), const_cast<float*>(lse), len_q, len_k, Tk};
    return from_hip(tsa::attn_bwd(x, as_rows(d_out, B, Hq, Tq), as_rows(dq, B, Hq, Tq), as_rows(dk, B, Hkv, Tk), as_rows(dv, B, Hkv, Tk),
                                  gate ? as_rows(dgate, B, Hq, Tq) : tsa::Rows16{nullptr, 0, 0, 0}, B, Hq, Hkv, Tq, D, scale, causal,
                                  ws, as_stream(stream)));
}
