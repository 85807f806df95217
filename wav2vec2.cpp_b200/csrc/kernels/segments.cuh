// Utterances as runs of packed rows (off[u] .. off[u]+T[u], off[u+1] >= off[u]+T[u]),
// and what the adapter kernels pass from the first product to the second.
#pragma once
#include "common.cuh"

namespace w2v {
namespace sg {

// The utterance that row r belongs to, or -1.
W2V_DEV int utterance_of(const long long* off, const int* T, int n_utt, long long r) {
    int lo = 0, hi = n_utt;      // first utterance that ends after r
    while (lo < hi) {
        const int m = (lo + hi) / 2;
        if (off[m] + max(T[m], 0) > r) hi = m; else lo = m + 1;
    }
    return lo < n_utt && off[lo] <= r ? lo : -1;
}

// Low-rank adapters: s_a A_a x of every row, laid out for a GEMM whose tiles
// take `tile` rows.  For each adapter that a tile's rows use there is a block
// [tile][rank] of fp16, zero in the rows of other adapters, so that the
// second product is (block) x (that adapter's B): further K-blocks of the
// tile's main product, however the tile's rows are spread over utterances.
// Tile i's blocks are first .. first + count - 1 with
//   first = i + min(utterances that start before the tile, rows before it),
// which leaves room for every tile without a scan over the tiles before: a
// tile has at most one utterance that started before it, and one per start in it.
struct LoraTile {
    int first, count;
};
struct LoraPlan {
    LoraTile* tiles;       // [row tiles]
    int* adapter;          // [blocks]
    __half* t;             // [parts][blocks][tile][rank]
    int tile;              // rows per tile: 64, 128, 192 or 256
    int rank;
    int parts;             // 1: fp16; 2: value and remainder (fp32 outputs)
    long long blocks;      // room for so many
};

struct LoraArgs {
    const __half* x;
    long long lda;
    int K;
    long long M;
    const __half* a;       // [n_adapters][rank][K]
    const float* scale;    // [n_adapters] or NULL
    int n_adapters;
    const long long* off;
    const int* T;
    const int* adapter;
    int n_utt;
};

__host__ inline long long lora_blocks(long long M, int n_utt, int tile) {
    return (M + tile - 1) / tile + (n_utt < M ? n_utt : M);
}
// Workspace for any tile height; lora_plan lays one height's plan out in it.
__host__ inline long long lora_workspace(long long M, int n_utt, int rank) {
    const long long rows = M + 256 * (1 + (n_utt < M ? n_utt : M));
    const long long tiles = M / 64 + 1;
    return (tiles * 8 + 255) / 256 * 256 + ((tiles + (n_utt < M ? n_utt : M)) * 4 + 255) / 256 * 256 + rows * rank * 4 + 256;
}
__host__ inline LoraPlan lora_plan(void* ws, long long M, int n_utt, int rank, int tile, int parts) {
    LoraPlan p;
    uint8_t* at = reinterpret_cast<uint8_t*>(ws);
    p.tile = tile;
    p.rank = rank;
    p.parts = parts;
    p.blocks = lora_blocks(M, n_utt, tile);
    p.tiles = reinterpret_cast<LoraTile*>(at);
    at += ((M + tile - 1) / tile * 8 + 255) / 256 * 256;
    p.adapter = reinterpret_cast<int*>(at);
    at += (p.blocks * 4 + 255) / 256 * 256;
    p.t = reinterpret_cast<__half*>(at);
    return p;
}

// Fills the plan: lora_shrink.cu.  The launch lets the next kernel of the
// stream start early; that one waits (grid_dependency_wait) before it reads the plan.
int lora_shrink(const LoraArgs& a, const LoraPlan& p, cudaStream_t st);

W2V_DEV void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
W2V_DEV void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace sg
}  // namespace w2v
