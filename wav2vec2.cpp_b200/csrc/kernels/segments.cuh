// Utterances as runs of packed rows (off[u] .. off[u]+T[u], off[u+1] >= off[u]+T[u]),
// and what the adapter kernels pass from the first product to the second.
#pragma once
#include "common.cuh"
#include "w2v_kernels.h"

namespace w2v {
namespace sg {

// Low-rank adapters: t = s_a A_a x of every row, laid out for a GEMM whose tiles
// take `tile` rows.  For each adapter that a tile's rows use there is a block
// of `tile` rows of fp16, zero in the rows of other adapters, so that the
// second product is (block) x (that adapter's B): further K-blocks of the
// tile's main product, however the tile's rows are spread over utterances.
//
// t is held as two fp16 numbers, the value and what its rounding left: 22 bits, as
// much as fp32 outputs need, and more than fp16 outputs can do without (with 11 bits
// they are off by half a step of their own in one place of three).  They stand side by side,
// 32 ranks of the one, then of the other, so that both meet the same columns of B within
// one K-block: a row is groups of 64 columns, the last of 2 w where w = 16 or 32 ranks
// are left (the rank rounded up to 16; zero behind it).
//
// A zero row times an infinity is no zero, so the blocks' zeros alone would let what one
// adapter's B holds reach every row of the tile: the block's owners are the rows that its
// product may change.
// Tile i's blocks are first .. first + count - 1 with
//   first = i + min(utterances that end before the tile, rows before it),
// which leaves room for every tile without a scan over the tiles before: of a
// tile's utterances all but one end in it.
constexpr int kInline = 14;
struct LoraTile {          // 64 bytes: one load of half a warp
    int first, count;
    int adapter[kInline];  // of the first blocks; those of the others in LoraPlan::adapter
};
struct LoraPlan {
    LoraTile* tiles;       // [row tiles]
    int* adapter;          // [blocks]
    uint32_t* owners;      // [blocks][kOwnerWords]: bit r % 32 of word r / 32, row r of the tile is this adapter's
    __half* t;             // [blocks][tile][t_columns(rank)]
    int tile;              // rows per tile: 64, 128, 192 or 256
    int rank;
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
    int* err;
    int sums;              // the sums over K end every 512 (fp32 outputs: segment_gemm.cu)
};

constexpr int kGroup = 32;                                                     // ranks whose values stand together
__host__ __device__ inline int rank16(int rank) { return (rank + 15) / 16 * 16; }
__host__ __device__ inline int t_columns(int rank) { return 2 * rank16(rank); }
// Ranks (rounded up to 16) of the group that begins at rank r.
__host__ __device__ inline int group_width(int rank, int r) { return rank16(rank) - r < kGroup ? rank16(rank) - r : kGroup; }

__host__ inline long long lora_blocks(long long M, int n_utt, int tile) {
    return (M + tile - 1) / tile + (n_utt < M ? n_utt : M);
}
constexpr int kOwnerWords = 8;               // 256 rows
// Workspace for any tile height; lora_plan lays one height's plan out in it.  -1: more rows
// of blocks than an int numbers (the TMA's coordinate).
__host__ inline long long lora_workspace(long long M, int n_utt, int rank) {
    const long long rows = M + 256 * (1 + (n_utt < M ? n_utt : M));
    if (rows > 0x7fffffffLL) return -1;
    const long long tiles = M / 64 + 1, blocks = tiles + (n_utt < M ? n_utt : M);
    return (tiles * (long long)sizeof(LoraTile) + 255) / 256 * 256 + (blocks * 4 + 255) / 256 * 256 +
           (blocks * kOwnerWords * 4 + 255) / 256 * 256 + rows * t_columns(rank) * 2 + 256;
}
__host__ inline LoraPlan lora_plan(void* ws, long long M, int n_utt, int rank, int tile) {
    LoraPlan p;
    uint8_t* at = reinterpret_cast<uint8_t*>(ws);
    p.tile = tile;
    p.rank = rank;
    p.blocks = lora_blocks(M, n_utt, tile);
    p.tiles = reinterpret_cast<LoraTile*>(at);
    at += ((M + tile - 1) / tile * (long long)sizeof(LoraTile) + 255) / 256 * 256;
    p.adapter = reinterpret_cast<int*>(at);
    at += (p.blocks * 4 + 255) / 256 * 256;
    p.owners = reinterpret_cast<uint32_t*>(at);
    at += (p.blocks * kOwnerWords * 4 + 255) / 256 * 256;
    p.t = reinterpret_cast<__half*>(at);
    return p;
}

// Fills the plan: lora_shrink.cu.  The launch lets the next kernel of the
// stream start early; that one waits (grid_dependency_wait) before it reads the plan.
// x: a map of the rows in boxes of x_rows, if the caller has one.
int lora_shrink(const LoraArgs& a, const LoraPlan& p, const CUtensorMap* x, int x_rows, cudaStream_t st);

inline PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        cudaDriverEntryPointQueryResult q;
        void* f = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
    }();
    return fn;
}

// fp16 [.., rows, inner] with 64 x `box_rows` boxes, 128-byte swizzle.
inline int map_f16(CUtensorMap* m, const void* base, int rank, const uint64_t* dims, const uint64_t* strides, int box_rows) {
    auto enc = get_encode();
    if (!enc) return W2V_ERR_DRIVER;
    const uint32_t box[4] = {64, (uint32_t)box_rows, 1, 1}, es[4] = {1, 1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base), dims, strides, box, es,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? W2V_OK
               : W2V_ERR_TENSOR_MAP;
}

// ── MMA issue from warp-uniform code ───────────────────────────────────────
// The whole warp runs the issuing loop and one elected lane's predicate guards
// the instructions: loop counters, descriptors and barriers then stay in
// uniform registers.  Under a branch on the lane the operands of every MMA have
// to be moved there first, some 200 cycles each, which bounds tiles of few columns.
// The whole warp's wait, with one answer for all lanes.
W2V_DEV bool mbar_wait_warp(uint64_t* bar, uint32_t parity, int* err) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}
// A value that all lanes hold, in a uniform register (the operands of a TMA load
// have to be there, and a value that came by a shuffle or from memory is not known to be).
W2V_DEV int uniform(int x) { return __reduce_max_sync(0xffffffffu, x); }
W2V_DEV uint64_t desc_plus(uint64_t desc, uint32_t bytes) { return desc + (bytes >> 4); }
template <bool PAIR>
W2V_DEV void umma_f16_if(uint32_t lead, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                         uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
            " @q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
            " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(lead)
            : "memory");
}
// The same, leaving the rows (TMEM lanes) whose bit is set as they are: words 0 .. 3 those of this
// CTA (the first of a pair), 4 .. 7 of the second.
template <bool PAIR>
W2V_DEV void umma_f16_masked_if(uint32_t lead, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                const uint32_t (&off)[kOwnerWords]) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred p, q;\n setp.eq.b32 p, 0, 0;\n setp.ne.b32 q, %4, 0;\n"
            " @q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8, %9, %10, %11, %12}, p;\n}" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(lead), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3]), "r"(off[4]),
            "r"(off[5]), "r"(off[6]), "r"(off[7])
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p, q;\n setp.eq.b32 p, 0, 0;\n setp.ne.b32 q, %4, 0;\n"
            " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n}" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(lead), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3])
            : "memory");
}
// bar: shared::cluster address
template <bool PAIR>
W2V_DEV void umma_commit_if(uint32_t lead, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
            " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar),
            "r"(lead)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
            " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar),
            "r"(lead)
            : "memory");
}

// TMA loads by the same scheme (some 450 cycles a stage of two loads otherwise).
// bar: shared::cluster address of the barrier that counts the bytes.
W2V_DEV void expect_tx_if(uint32_t lead, uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
        " @q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}" ::"r"(bar),
        "r"(bytes), "r"(lead)
        : "memory");
}
// Bytes to come in the current phase, without an arrival.
W2V_DEV void expect_more_if(uint32_t lead, uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
        " @q mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n}" ::"r"(bar),
        "r"(bytes), "r"(lead)
        : "memory");
}
template <bool PAIR>
W2V_DEV void tma_load_2d_if(uint32_t lead, uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %5, 0;\n"
            " @q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4}], [%2];\n}" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(lead)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %5, 0;\n"
            " @q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4}], [%2];\n}" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(lead)
            : "memory");
}
template <bool PAIR>
W2V_DEV void tma_load_3d_if(uint32_t lead, uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1, int c2) {
    if constexpr (PAIR)
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %6, 0;\n"
            " @q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5}], [%2];\n}" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(lead)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred q;\n setp.ne.b32 q, %6, 0;\n"
            " @q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5}], [%2];\n}" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(lead)
            : "memory");
}

W2V_DEV void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
W2V_DEV void grid_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace sg
}  // namespace w2v
