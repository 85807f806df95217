// Products whose weights depend on the row's utterance: low-rank adapters
// beside a shared projection, and weight matrices per group of utterances.
//
//   lora     y[r] = epi(W x[r] + bias + s_a B_a (A_a x[r])),  a = adapter of r's utterance
//   grouped  y[r] = epi(W_g x[r] + bias_g),                   g = group of r's utterance
//
// 64 x 64 output tiles per block of 256 threads, operands through shared
// memory as fp32, 4 x 4 outputs per thread on the FMA pipes.
#include "common.cuh"
#include "w2v_kernels.h"

namespace w2v {
namespace sg {

constexpr int kTile = 64, kStep = 16;
enum : int { kF16 = 0, kQ8 = 1, kQ4 = 2 };

struct Params {
    const __half* A;
    long long lda;
    int K, N;
    long long M;
    const void* W;
    const __half* scales;
    long long ld_s;
    void* C;
    long long ldc;
    const float* bias;
    const float* resid;
    long long ldr;
    int epilogue;
    const long long* off;
    const int* T;
    const int* index;       // adapter or group of each utterance
    int n_utt, n_index;
    const __half* la;
    const __half* lb;
    const float* lscale;
    int rank;
    float* t;               // [M][rank] s_a A_a x
};

// The utterance that row r belongs to (off[u + 1] >= off[u] + T[u]), or -1.
W2V_DEV int utterance_of(const long long* off, const int* T, int n_utt, long long r) {
    int lo = 0, hi = n_utt;      // first utterance that ends after r
    while (lo < hi) {
        const int m = (lo + hi) / 2;
        if (off[m] + max(T[m], 0) > r) hi = m; else lo = m + 1;
    }
    return lo < n_utt && off[lo] <= r ? lo : -1;
}
W2V_DEV int index_of(const Params& p, long long r) {
    const int u = utterance_of(p.off, p.T, p.n_utt, r);
    if (u < 0) return -1;
    const int a = p.index[u];
    return a >= 0 && a < p.n_index ? a : -1;
}

template <int WQ>
W2V_DEV float weight(const Params& p, long long row, int n, int k) {
    if (WQ == kF16) return __half2float(reinterpret_cast<const __half*>(p.W)[row * p.K + k]);
    const __half d = p.scales[(k / 32) * p.ld_s + n];
    int q;
    if (WQ == kQ8) q = reinterpret_cast<const int8_t*>(p.W)[row * p.K + k];
    else {
        const uint32_t w = reinterpret_cast<const uint32_t*>(p.W)[row * (p.K / 8) + k / 8];
        const int j = k & 7;
        q = (int)(w >> (4 * (j >> 1) + 16 * (j & 1)) & 15u) - 8;
    }
    return __half2float(__hmul(__int2half_rn(q), d));   // d * q rounded once
}

// t[r] = s_a A_a x[r]: one warp per row.
__global__ void shrink_kernel(Params p) {
    const long long r = blockIdx.x * 8LL + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (r >= p.M) return;
    const int a = index_of(p, r);
    const float s = a < 0 ? 0.f : p.lscale ? p.lscale[a] : 1.f;
    for (int j = 0; j < p.rank; j++) {
        float acc = 0.f;
        if (a >= 0)
            for (int k = lane; k < p.K; k += 32)
                acc += __half2float(p.A[r * p.lda + k]) * __half2float(p.la[((long long)a * p.rank + j) * p.K + k]);
        for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
        if (lane == 0) p.t[r * p.rank + j] = acc * s;
    }
}

template <int WQ, bool GROUPED>
__global__ void __launch_bounds__(256) tile_kernel(Params p) {
    __shared__ float sx[kStep][kTile + 4], sw[kStep][kTile + 4];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int n0 = blockIdx.x * kTile;
    long long r0 = blockIdx.y * (long long)kTile, r1 = p.M;
    long long wrow = 0;
    int g = 0;
    if (GROUPED) {
        const int u = blockIdx.z;
        g = p.index[u];
        if (g < 0 || g >= p.n_index) return;
        r1 = min(p.M, p.off[u] + max(p.T[u], 0));
        r0 += p.off[u];
        wrow = (long long)g * p.N;
    }
    if (r0 >= r1) return;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += kStep) {
        for (int i = tid; i < kTile * kStep; i += 256) {
            const int k = i % kStep, m = i / kStep;
            sx[k][m] = r0 + m < r1 ? __half2float(p.A[(r0 + m) * p.lda + k0 + k]) : 0.f;
            sw[k][m] = n0 + m < p.N ? weight<WQ>(p, wrow + n0 + m, n0 + m, k0 + k) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kStep; k++) {
            float x[4], w[4];
            for (int i = 0; i < 4; i++) { x[i] = sx[k][ty * 4 + i]; w[i] = sw[k][tx * 4 + i]; }
            for (int i = 0; i < 4; i++)
                for (int j = 0; j < 4; j++) acc[i][j] += x[i] * w[j];
        }
        __syncthreads();
    }
    for (int i = 0; i < 4; i++) {
        const long long r = r0 + ty * 4 + i;
        if (r >= r1) continue;
        const int a = GROUPED ? -1 : index_of(p, r);
        for (int j = 0; j < 4; j++) {
            const int n = n0 + tx * 4 + j;
            if (n >= p.N) continue;
            float y = acc[i][j];
            if (a >= 0) {
                const __half* b = p.lb + ((long long)a * p.N + n) * p.rank;
                for (int q = 0; q < p.rank; q++) y += p.t[r * p.rank + q] * __half2float(b[q]);
            }
            if (p.bias) y += p.bias[(long long)g * p.N + n];
            if (p.epilogue == W2V_EPI_F16_GELU) y = gelu_tanh(y);
            if (p.epilogue == W2V_EPI_F32_RESID) y += p.resid[r * p.ldr + n];
            if (p.epilogue == W2V_EPI_F16 || p.epilogue == W2V_EPI_F16_GELU)
                reinterpret_cast<__half*>(p.C)[r * p.ldc + n] = __float2half_rn(y);
            else
                reinterpret_cast<float*>(p.C)[r * p.ldc + n] = y;
        }
    }
}

static bool bad_common(const Params& p) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p.A), w = reinterpret_cast<uintptr_t>(p.W);
    if (p.K <= 0 || p.K % 64 || p.M < 0 || p.M > 0x7fffffffLL || p.N <= 0 || p.lda < p.K || p.lda % 8 || p.ldc < p.N ||
        ((a | w) & 15) || p.epilogue < W2V_EPI_F16 || p.epilogue > W2V_EPI_F32_RESID || p.n_utt < 0)
        return true;
    return p.M > 0 && (!p.A || !p.W || !p.C || (p.epilogue == W2V_EPI_F32_RESID && (!p.resid || p.ldr < p.N)) ||
                       (p.n_utt > 0 && (!p.off || !p.T || !p.index)));
}

static int lora(Params p, int wq, const void* lora_a, const void* lora_b, const float* lora_scale, int n_adapters,
                int rank, void* workspace, long long workspace_bytes, cudaStream_t st) {
    if (bad_common(p) || rank < 8 || rank > 128 || rank % 8 || n_adapters <= 0 || !lora_a || !lora_b ||
        ((reinterpret_cast<uintptr_t>(lora_a) | reinterpret_cast<uintptr_t>(lora_b)) & 15))
        return W2V_ERR_ARGS;
    if (p.M == 0) return W2V_OK;
    const long long need = w2v_lora_workspace_bytes(p.M, p.n_utt, rank);
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 127)) return W2V_ERR_ARGS;
    if (workspace_bytes < need) return W2V_ERR_CAPACITY;
    p.la = reinterpret_cast<const __half*>(lora_a);
    p.lb = reinterpret_cast<const __half*>(lora_b);
    p.lscale = lora_scale;
    p.n_index = n_adapters;
    p.rank = rank;
    p.t = reinterpret_cast<float*>(workspace);
    shrink_kernel<<<(unsigned)((p.M + 7) / 8), 256, 0, st>>>(p);
    const dim3 grid((p.N + kTile - 1) / kTile, (unsigned)((p.M + kTile - 1) / kTile));
    if (wq == kF16) tile_kernel<kF16, false><<<grid, 256, 0, st>>>(p);
    else if (wq == kQ8) tile_kernel<kQ8, false><<<grid, 256, 0, st>>>(p);
    else tile_kernel<kQ4, false><<<grid, 256, 0, st>>>(p);
    return cudaPeekAtLastError() == cudaSuccess ? W2V_OK : W2V_ERR_LAUNCH;
}

}  // namespace sg
}  // namespace w2v

using namespace w2v::sg;

extern "C" long long w2v_lora_workspace_bytes(long long M, int n_utt, int rank) {
    if (M < 0 || n_utt < 0 || rank < 8 || rank > 128 || rank % 8) return -1;
    return (M * rank * 4 + 127) / 128 * 128;
}

extern "C" int w2v_gemm_f16_lora(const void* A, long long lda, long long K, long long M, const void* B, int N, void* C,
                                 long long ldc, const float* bias, const float* resid, long long ldr, int epilogue,
                                 const void* lora_a, const void* lora_b, const float* lora_scale, int n_adapters,
                                 int rank, const long long* off, const int* T, const int* adapter, int n_utt,
                                 void* workspace, long long workspace_bytes, int* err, void* stream) {
    if (K > 0x7fffffffLL) return W2V_ERR_ARGS;
    Params p = {};
    p.A = reinterpret_cast<const __half*>(A); p.lda = lda; p.K = (int)K; p.M = M; p.W = B; p.N = N; p.C = C;
    p.ldc = ldc; p.bias = bias; p.resid = resid; p.ldr = ldr; p.epilogue = epilogue;
    p.off = off; p.T = T; p.index = adapter; p.n_utt = n_utt;
    return lora(p, kF16, lora_a, lora_b, lora_scale, n_adapters, rank, workspace, workspace_bytes,
                reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int w2v_gemm_q_lora(const void* A, long long lda, long long K, long long M, const void* Bq, const void* Bs,
                               long long ld_s, int gguf_type, int N, void* C, long long ldc, const float* bias,
                               const float* resid, long long ldr, int epilogue, const void* lora_a,
                               const void* lora_b, const float* lora_scale, int n_adapters, int rank,
                               const long long* off, const int* T, const int* adapter, int n_utt, void* workspace,
                               long long workspace_bytes, int* err, void* stream) {
    const int wq = gguf_type == 8 ? kQ8 : gguf_type == 2 ? kQ4 : 0;
    if (!wq || K > 0x7fffffffLL || !Bs || (reinterpret_cast<uintptr_t>(Bs) & 15) || ld_s < N || ld_s % 8)
        return W2V_ERR_ARGS;
    Params p = {};
    p.A = reinterpret_cast<const __half*>(A); p.lda = lda; p.K = (int)K; p.M = M; p.W = Bq; p.N = N; p.C = C;
    p.scales = reinterpret_cast<const __half*>(Bs); p.ld_s = ld_s;
    p.ldc = ldc; p.bias = bias; p.resid = resid; p.ldr = ldr; p.epilogue = epilogue;
    p.off = off; p.T = T; p.index = adapter; p.n_utt = n_utt;
    return lora(p, wq, lora_a, lora_b, lora_scale, n_adapters, rank, workspace, workspace_bytes,
                reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int w2v_gemm_grouped_f16(const void* A, long long lda, long long K, long long M, const void* B,
                                    int n_groups, int N, void* C, long long ldc, const float* bias,
                                    const float* resid, long long ldr, int epilogue, const long long* off,
                                    const int* T, const int* group, int n_utt, int* err, void* stream) {
    if (K > 0x7fffffffLL || n_groups <= 0) return W2V_ERR_ARGS;
    Params p = {};
    p.A = reinterpret_cast<const __half*>(A); p.lda = lda; p.K = (int)K; p.M = M; p.W = B; p.N = N; p.C = C;
    p.ldc = ldc; p.bias = bias; p.resid = resid; p.ldr = ldr; p.epilogue = epilogue;
    p.off = off; p.T = T; p.index = group; p.n_index = n_groups; p.n_utt = n_utt;
    if (bad_common(p)) return W2V_ERR_ARGS;
    if (M == 0 || n_utt == 0) return W2V_OK;
    if (n_utt > 65535) return W2V_ERR_CAPACITY;
    const dim3 grid((N + kTile - 1) / kTile, (unsigned)((M + kTile - 1) / kTile), n_utt);
    tile_kernel<kF16, true><<<grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
    return cudaPeekAtLastError() == cudaSuccess ? W2V_OK : W2V_ERR_LAUNCH;
}
