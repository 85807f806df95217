// Low-rank adapters beside a projection on Q8_0 / Q4_0 weights: the
// dequant-fused GEMM with the adapters' k-blocks behind the main ones
// (qgemm_tc.cuh, segments.cuh).
#include "qgemm_tc.cuh"

namespace w2v {
namespace qg {

// Tiles whose heights in activation rows are multiples of the 64 rows that a
// block of the first product covers.
static int pick_lora_tile(int N, int m_valid) {
    const int sms = sm_count();
    int best = 128;
    double best_cost = 1e300;
    for (int bn : {-192, -128, 128, 64}) {
        const bool pair = bn < 0;
        const int w = pair ? -bn : bn;
        const long long ft = (N + kRows * (pair ? 2 : 1) - 1) / (kRows * (pair ? 2 : 1));
        const long long rt = (m_valid + w - 1) / w;
        const long long slots = pair ? sms / 2 : sms;
        const long long waves = (ft * rt + slots - 1) / slots;
        const double cost = (double)waves * w * tile_row_cost(bn);
        if (cost < best_cost) { best_cost = cost; best = bn; }
    }
    return best;
}

// Two epilogue warps per lane quarter for the heavier epilogues, as without adapters (launch_w).
template <int EPI, int WQ>
static int launch_lora(int bn, const QMaps& m, const QParams& p, const QLora<true>& lo, cudaStream_t st) {
    constexpr int EH = EPI == W2V_EPI_F16 ? 1 : 2;
    switch (bn) {
        case -192: return launch<192, EPI, WQ, true, EH, true>(m.x, m.q, m.s, m.c, m.r, p, st, lo);
        case -128: return launch<128, EPI, WQ, true, EH, true>(m.x, m.q, m.s, m.c, m.r, p, st, lo);
        case 128: return launch<128, EPI, WQ, false, EH, true>(m.x, m.q, m.s, m.c, m.r, p, st, lo);
        default: return launch<64, EPI, WQ, false, EH, true>(m.x, m.q, m.s, m.c, m.r, p, st, lo);
    }
}

template <int EPI>
static int launch_lora_w(int wq, int bn, const QMaps& m, const QParams& p, const QLora<true>& lo, cudaStream_t st) {
    return wq == kQ8 ? launch_lora<EPI, kQ8>(bn, m, p, lo, st) : launch_lora<EPI, kQ4>(bn, m, p, lo, st);
}

}  // namespace qg
}  // namespace w2v

using namespace w2v;
using namespace w2v::qg;

extern "C" int w2v_gemm_q_lora(const void* A, long long lda, long long K, long long M, const void* Bq, const void* Bs,
                               long long ld_s, int gguf_type, int N, void* C, long long ldc, const float* bias,
                               const float* resid, long long ldr, int epilogue, const void* lora_a,
                               const void* lora_b, const float* lora_scale, int n_adapters, int rank,
                               const long long* off, const int* T, const int* adapter, int n_utt, void* workspace,
                               long long workspace_bytes, int* err, void* stream) {
    if (lda < K || lda % 8 || rank < 8 || rank > 128 || rank % 8 || n_adapters <= 0 || !lora_a || !lora_b ||
        ((reinterpret_cast<uintptr_t>(lora_a) | reinterpret_cast<uintptr_t>(lora_b)) & 15) || n_utt < 0 ||
        M > 0x7fffffffLL - 512 || N > 0x7fffffff - 512 || n_utt > 0x7fffffff - 512 || epilogue == W2V_EPI_F32_RESID_LN || !Bq || !Bs || K > 0x7fffffffLL)
        return W2V_ERR_ARGS;
    if (M == 0 && K > 0 && K % kBK == 0 && N > 0 && ldc >= N) return W2V_OK;
    if (n_utt > 0 && (!off || !T || !adapter)) return W2V_ERR_ARGS;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 127)) return W2V_ERR_ARGS;
    if (M < 0) return W2V_ERR_ARGS;
    const long long need = sg::lora_workspace(M, n_utt, rank);
    if (need < 0) return W2V_ERR_ARGS;
    if (workspace_bytes < need) return W2V_ERR_CAPACITY;
    QParams p;
    QMaps m;
    int bn = 0;
    int rc = qgemm_setup(A, lda, K, M, Bq, Bs, ld_s, gguf_type, N, C, ldc, bias, resid, ldr, epilogue, nullptr, nullptr,
                         nullptr, 0, err, pick_lora_tile, p, m, &bn);
    if (rc || !bn) return rc;
    const int wq = gguf_type == 8 ? kQ8 : kQ4;
    const int rows = bn < 0 ? -bn : bn;
    const bool f16 = epilogue == W2V_EPI_F16 || epilogue == W2V_EPI_F16_GELU;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    QLora<true> lo;
    lo.t = lo.b = m.x;
    lo.lora = n_utt > 0;
    lo.lb = reinterpret_cast<const __half*>(lora_b);
    lo.plan = sg::lora_plan(workspace, M, n_utt, rank, rows);
    // as the fp16 kernel does (segment_gemm.cu): 512 of K, 1024 beside a residual
    lo.sum_blocks = epilogue == W2V_EPI_F32_RESID ? 16 : 8;
    lo.n_sums = f16 ? 1 : (int)((K / kBK + lo.sum_blocks - 1) / lo.sum_blocks);
    lo.chunks = (2 * rank + code_row_bytes(wq) - 1) / code_row_bytes(wq);
    if (lo.lora) {
        auto enc = get_encode();
        const uint32_t es[3] = {1, 1, 1};
        const uint64_t td[2] = {(uint64_t)sg::t_columns(rank), (uint64_t)(lo.plan.blocks * rows)};
        const uint64_t ts[1] = {(uint64_t)sg::t_columns(rank) * 2};
        const uint32_t tbox[2] = {kBK, (uint32_t)(bn < 0 ? rows / 2 : rows)};
        if (enc(&lo.t, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, lo.plan.t, td, ts, tbox, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return W2V_ERR_TENSOR_MAP;
        const uint64_t bd[3] = {(uint64_t)rank * 2, (uint64_t)N, (uint64_t)n_adapters};
        const uint64_t bs[2] = {(uint64_t)rank * 2, (uint64_t)rank * 2 * N};
        const uint32_t bbox[3] = {(uint32_t)code_row_bytes(wq), (uint32_t)kRows, 1};
        if (enc(&lo.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(lora_b), bd, bs, bbox, es,
                CU_TENSOR_MAP_INTERLEAVE_NONE, wq == kQ8 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return W2V_ERR_TENSOR_MAP;
        const sg::LoraArgs a{reinterpret_cast<const __half*>(A), lda, (int)K, M, reinterpret_cast<const __half*>(lora_a),
                             lora_scale, n_adapters, off, T, adapter, n_utt, err, !f16};
        rc = sg::lora_shrink(a, lo.plan, nullptr, 0, st);
        if (rc) return rc;
    }
    switch (epilogue) {
        case W2V_EPI_F16: return launch_lora_w<W2V_EPI_F16>(wq, bn, m, p, lo, st);
        case W2V_EPI_F16_GELU: return launch_lora_w<W2V_EPI_F16_GELU>(wq, bn, m, p, lo, st);
        case W2V_EPI_F32: return launch_lora_w<W2V_EPI_F32>(wq, bn, m, p, lo, st);
        default: return launch_lora_w<W2V_EPI_F32_RESID>(wq, bn, m, p, lo, st);
    }
}
