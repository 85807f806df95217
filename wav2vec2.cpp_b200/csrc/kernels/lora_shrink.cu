// First product of the low-rank adapters: t = s_a A_a x for every row, written
// as the masked fp16 blocks that the projections add as further K-blocks
// (segments.cuh).
//
// 2 M K rank operations on M K fp16 values: with the ranks in use (8 .. 128)
// the read of x bounds it.  A block of 128 threads takes 64 rows (of one row
// tile) and K in steps of 64 through a ring of shared-memory stages filled by
// cp.async; each warp multiplies 16 rows by all `rank` rows of A_a with
// m16n8k16 instructions, fp32 accumulators in registers.  Several blocks per
// SM keep some 100 KB of x in flight.  A row tile used by several adapters is
// done once per adapter, by blockIdx.y in turn, where any of the 64 rows use it.
#include "segments.cuh"
#include "w2v_kernels.h"

namespace w2v {
namespace sg {

constexpr int kRows = 64, kStep = 64, kThreads = 128, kMaxTile = 256;

__host__ __device__ constexpr int stage_bytes(int rank) { return (kRows + rank) * kStep * 2; }

// 16-byte group g of row r of a [rows][64] fp16 tile, 128-byte rows, groups
// XOR-swizzled by row so that both the copies and ldmatrix are conflict free.
W2V_DEV uint32_t tile_at(uint32_t base, int r, int g) { return base + (uint32_t)(r * 128 + ((g ^ (r & 7)) << 4)); }

W2V_DEV void cp_async16_zfill(uint32_t saddr, const void* g, bool real) {
    const int n = real ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(saddr), "l"(g), "r"(n) : "memory");
}

template <int NT>   // rank / 8
__global__ void __launch_bounds__(kThreads) lora_shrink_kernel(LoraArgs a, LoraPlan p, int stages) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int row_adapter[kMaxTile];
    __shared__ int slots[kMaxTile];           // the tile's adapters, by their first row
    __shared__ int n_slots;
    constexpr int rank = NT * 8;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    grid_launch_dependents();
    const long long row0 = (long long)blockIdx.x * kRows;
    const long long tile = row0 / p.tile;
    const long long tile0 = tile * p.tile;
    const int n_rows = (int)min((long long)p.tile, a.M - tile0);

    // adapters of the tile's rows
    auto adapter_of = [&](int u) {
        const int v = u < 0 ? -1 : a.adapter[u];
        return v >= 0 && v < a.n_adapters ? v : -1;
    };
    for (int i = tid; i < n_rows; i += kThreads)
        row_adapter[i] = adapter_of(utterance_of(a.off, a.T, a.n_utt, tile0 + i));
    if (tid == 0) n_slots = 0;
    __syncthreads();
    for (int i0 = 0; i0 < n_rows; i0 += kThreads) {
        const int i = i0 + tid;
        bool first = false;
        if (i < n_rows) {
            const int v = row_adapter[i];
            first = v >= 0 && (i == 0 || row_adapter[i - 1] != v);
            for (int j = 0; first && j < i; j++) first = row_adapter[j] != v;
        }
        __shared__ int base[kThreads / 32];
        const uint32_t m = __ballot_sync(0xffffffffu, first);
        if (lane == 0) base[warp] = __popc(m);
        __syncthreads();
        int at = n_slots;
        for (int w = 0; w < warp; w++) at += base[w];
        if (first) slots[at + __popc(m & ((1u << lane) - 1u))] = row_adapter[i];
        __syncthreads();
        if (tid == kThreads - 1) n_slots = at + __popc(m);
        __syncthreads();
    }
    const int count = n_slots;
    // first block of the tile
    int lo = 0, hi = a.n_utt;                 // utterances that start before the tile
    while (lo < hi) {
        const int m = (lo + hi) / 2;
        if (a.off[m] < tile0) lo = m + 1; else hi = m;
    }
    const long long first_block = tile + (lo < tile0 ? lo : tile0);
    if (row0 == tile0 && blockIdx.y == 0) {
        if (tid == 0) p.tiles[tile] = LoraTile{(int)first_block, count};
        for (int i = tid; i < count; i += kThreads) p.adapter[first_block + i] = slots[i];
    }

    const int k_steps = a.K / kStep;
    const uint32_t sbase = smem_u32(smem);
    const int local0 = (int)(row0 - tile0);
    for (int s = blockIdx.y; s < count; s += gridDim.y) {
        const int ad = slots[s];
        bool mine = false;                    // any of the 64 rows
        if (tid < kRows && local0 + tid < n_rows) mine = row_adapter[local0 + tid] == ad;
        const bool some = __syncthreads_or(mine);
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[n][i] = 0.f;
        if (some) {
            const __half* wa = a.a + (long long)ad * rank * a.K;
            auto fetch = [&](int ks) {
                const uint32_t st = sbase + (uint32_t)((ks % stages) * stage_bytes(rank));
                const int k0 = ks * kStep;
#pragma unroll
                for (int i = 0; i < kRows * 8 / kThreads; i++) {
                    const int c = tid + i * kThreads, r = c >> 3, g = c & 7;
                    const bool real = row0 + r < a.M;
                    cp_async16_zfill(tile_at(st, r, g), a.x + (real ? row0 + r : 0) * a.lda + k0 + g * 8, real);
                }
                for (int c = tid; c < rank * 8; c += kThreads) {
                    const int r = c >> 3, g = c & 7;
                    cp_async16(tile_at(st + kRows * kStep * 2, r, g), wa + (long long)r * a.K + k0 + g * 8);
                }
            };
            for (int ks = 0; ks < stages - 1; ks++) {
                if (ks < k_steps) fetch(ks);
                cp_async_commit();
            }
            for (int ks = 0; ks < k_steps; ks++) {
                // stage ks has landed when at most stages - 2 younger groups are under way
                if (stages == 4) cp_async_wait<2>(); else cp_async_wait<1>();
                __syncthreads();
                if (ks + stages - 1 < k_steps) fetch(ks + stages - 1);
                cp_async_commit();
                const uint32_t sx = sbase + (uint32_t)((ks % stages) * stage_bytes(rank)), sa = sx + kRows * kStep * 2;
#pragma unroll
                for (int kk = 0; kk < 4; kk++) {
                    uint32_t x0, x1, x2, x3;
                    ldsm_x4(tile_at(sx, warp * 16 + (lane & 15), kk * 2 + (lane >> 4)), x0, x1, x2, x3);
#pragma unroll
                    for (int n = 0; n < NT; n += 2) {
                        uint32_t b0, b1, b2, b3;   // ranks 8n .. 8n+7 (k low, k high), then 8n+8 .. (the last odd one twice)
                        const int r = n + 1 < NT ? n * 8 + (lane & 7) + ((lane >> 4) << 3) : n * 8 + (lane & 7);
                        ldsm_x4(tile_at(sa, r, kk * 2 + ((lane >> 3) & 1)), b0, b1, b2, b3);
                        mma_16816(acc[n], x0, x1, x2, x3, b0, b1);
                        if (n + 1 < NT) mma_16816(acc[n + 1], x0, x1, x2, x3, b2, b3);
                    }
                }
            }
            cp_async_wait<0>();
        }
        // masked, as fp16 (and what the rounding left, for fp32 outputs)
        const float sc = a.scale ? a.scale[ad] : 1.f;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = local0 + warp * 16 + (lane >> 2) + 8 * h;
            if (r >= n_rows) continue;
            const bool on = row_adapter[r] == ad;
            __half* out = p.t + ((first_block + s) * p.tile + r) * rank + (lane & 3) * 2;
            const long long part = p.blocks * p.tile * rank;
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float v0 = on ? acc[n][2 * h] * sc : 0.f, v1 = on ? acc[n][2 * h + 1] * sc : 0.f;
                const __half2 hi = __floats2half2_rn(v0, v1);
                *reinterpret_cast<__half2*>(out + n * 8) = hi;
                if (p.parts == 2) {
                    const float2 f = __half22float2(hi);
                    const float l0 = isinf(f.x) ? 0.f : v0 - f.x, l1 = isinf(f.y) ? 0.f : v1 - f.y;
                    *reinterpret_cast<__half2*>(out + part + n * 8) = __floats2half2_rn(l0, l1);
                }
            }
        }
        __syncthreads();       // the stages are read before the next adapter's copies
    }
}

template <int NT>
static int launch_nt(const LoraArgs& a, const LoraPlan& p, cudaStream_t st) {
    const int stages = stage_bytes(NT * 8) * 4 <= 64 * 1024 ? 4 : 3;
    const int smem = stages * stage_bytes(NT * 8);
    auto kern = lora_shrink_kernel<NT>;
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!attr_set[dev & 63]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return W2V_ERR_LAUNCH;
        attr_set[dev & 63] = true;
    }
    // few row chunks: as many blocks per chunk as adapters can meet there, so that they run side by side
    const long long chunks = (a.M + kRows - 1) / kRows;
    long long most = p.tile;
    if (a.n_utt < most) most = a.n_utt;
    if (a.n_adapters < most) most = a.n_adapters;
    long long ny = 296 / chunks;
    ny = ny < 1 ? 1 : ny > most ? most : ny;
    kern<<<dim3((unsigned)chunks, (unsigned)ny), kThreads, smem, st>>>(a, p, stages);
    return cudaPeekAtLastError() == cudaSuccess ? W2V_OK : W2V_ERR_LAUNCH;
}

int lora_shrink(const LoraArgs& a, const LoraPlan& p, cudaStream_t st) {
    switch (p.rank / 8) {
#define W2V_SHRINK(n) case n: return launch_nt<n>(a, p, st);
        W2V_SHRINK(1) W2V_SHRINK(2) W2V_SHRINK(3) W2V_SHRINK(4) W2V_SHRINK(5) W2V_SHRINK(6) W2V_SHRINK(7) W2V_SHRINK(8)
        W2V_SHRINK(9) W2V_SHRINK(10) W2V_SHRINK(11) W2V_SHRINK(12) W2V_SHRINK(13) W2V_SHRINK(14) W2V_SHRINK(15) W2V_SHRINK(16)
#undef W2V_SHRINK
        default: return W2V_ERR_ARGS;
    }
}

}  // namespace sg
}  // namespace w2v
