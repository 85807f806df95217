// Entry points of the dequant-fused GEMM (qgemm_tc.cuh).
#include "qgemm_tc.cuh"

namespace w2v {
namespace qg {

static int qgemm_impl(const void* A, long long K, long long M, const void* Bq, const void* Bs, long long ld_s,
                      int gguf_type, int N, void* C, long long ldc, const float* bias, const float* resid,
                      long long ldr, int epilogue, const float* ln_stats, const float* ln_w, const float* ln_b,
                      int block_n, int* err, void* stream) {
    QParams p;
    QMaps m;
    int bn = 0;
    const int rc = qgemm_setup(A, K, K, M, Bq, Bs, ld_s, gguf_type, N, C, ldc, bias, resid, ldr, epilogue, ln_stats, ln_w,
                               ln_b, block_n, err, pick_tile, p, m, &bn);
    if (rc || !bn) return rc;
    const int wq = gguf_type == 8 ? kQ8 : kQ4;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int eh = p.tma ? 2 : 1;   // used by the residual and GELU epilogues (launch_w)
    switch (epilogue) {
        case W2V_EPI_F16: return launch_w<W2V_EPI_F16>(wq, bn, 1, m.x, m.q, m.s, m.c, m.r, p, st);
        case W2V_EPI_F16_GELU: return launch_w<W2V_EPI_F16_GELU>(wq, bn, eh, m.x, m.q, m.s, m.c, m.r, p, st);
        case W2V_EPI_F32: return launch_w<W2V_EPI_F32>(wq, bn, 1, m.x, m.q, m.s, m.c, m.r, p, st);
        case W2V_EPI_F32_RESID: return launch_w<W2V_EPI_F32_RESID>(wq, bn, eh, m.x, m.q, m.s, m.c, m.r, p, st);
        default: return launch_w<W2V_EPI_F32_RESID_LN>(wq, bn, eh, m.x, m.q, m.s, m.c, m.r, p, st);
    }
}

}  // namespace qg
}  // namespace w2v

extern "C" int w2v_gemm_q(const void* A, long long K, long long M, const void* Bq, const void* Bs, long long ld_s,
                          int gguf_type, int N, void* C, long long ldc, const float* bias, const float* resid,
                          long long ldr, int epilogue, int block_n, int* err, void* stream) {
    if (epilogue == W2V_EPI_F32_RESID_LN) return W2V_ERR_ARGS;   // needs the statistics: w2v_gemm_q_ln_resid
    return w2v::qg::qgemm_impl(A, K, M, Bq, Bs, ld_s, gguf_type, N, C, ldc, bias, resid, ldr, epilogue, nullptr,
                               nullptr, nullptr, block_n, err, stream);
}

extern "C" int w2v_gemm_q_ln_resid(const void* A, long long K, long long M, const void* Bq, const void* Bs,
                                   long long ld_s, int gguf_type, int N, void* C, long long ldc, const float* bias,
                                   const float* resid, long long ldr, const float* ln_stats, const float* ln_w,
                                   const float* ln_b, int block_n, int* err, void* stream) {
    return w2v::qg::qgemm_impl(A, K, M, Bq, Bs, ld_s, gguf_type, N, C, ldc, bias, resid, ldr, W2V_EPI_F32_RESID_LN,
                               ln_stats, ln_w, ln_b, block_n, err, stream);
}
