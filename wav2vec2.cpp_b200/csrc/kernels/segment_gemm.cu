// Products whose weights depend on the row's utterance, on fp16 weights:
//
//   lora     y[r] = epi(W x[r] + bias + s_a B_a (A_a x[r])),  a = adapter of r's utterance
//   grouped  y[r] = epi(W_g x[r] + bias_g),                   g = group of r's utterance
//
// One persistent warp-specialised tcgen05 kernel serves both: TMA-fed 128-byte
// swizzled operand tiles, fp32 accumulators in TMEM (two, so that the
// epilogue of a tile overlaps the products of the next), single CTAs on
// 128-row tiles or CTA pairs (cta_group::2) on 256-row tiles.  The tile width
// is a launch parameter (any multiple of 32 up to 256: the MMA's N, the
// weight box and the number of stages follow from it), so that narrow
// outputs such as a head of 200 tokens do not pay for 256 columns.
//
// lora: tiles cover the packed rows as those of w2v_gemm_f16 do.  The adapters
// are further K-blocks of the same accumulation: the first product (s_a A_a x,
// lora_shrink.cu) lies in blocks of a tile's rows, one per adapter among them and
// zero in the other rows, and is multiplied by that adapter's B.  The delta
// thus costs rank / K of the main product per adapter in the tile, is added
// in fp32 before the only rounding, and needs no pass of its own over y.  The
// kernel starts while the first product runs and waits for it only before the
// last K-block of its first tile.
//
// fp32 outputs: the tensor core's accumulation drops what lies behind the 24th bit
// of each partial sum, always towards zero, which over K = 1024 adds up to 1.2e-6 of
// the result.  For them an accumulator is handed over every 512 of K (beside a residual:
// 1024), the epilogue warps add it, rounding to nearest, to a running total that has
// columns of its own in TMEM, and the error stays that of some 32 steps at any K
// (4.6e-7 on normal inputs, with adapters, whose first product is summed alike, 5.6e-7).  The MMAs wait for the hand-over where the tile leaves no room for a
// second accumulator (more than 160 columns): 38663 rows of 1024 x 200 take 34 us,
// with fp16 outputs 24.  (Totals in registers: 56, the epilogue then spills.)
//
// grouped: tiles are cut utterance by utterance (a warp-wide walk over the
// utterances' lengths finds each tile, in order, so nothing is planned on the
// host and no workspace is needed); rows past the utterance are computed and
// not stored.
//
// Bound: many rows by the MMAs (the tensor pipe is busy 72 to 85 % of the cycles, the ways
// from L2 at 38 to 42 % of their peak), few rows by the launches and the dependent waits.
// From a short graph (in brackets: call after call for some time, at the clock that the power
// limit then leaves, or the host's issue): 31936 rows, K 768, N 2304, rank 16: 105 us (125),
// 1.10 PFLOP/s; 31.7 K rows, 1024 x 4096, rank 32, GELU: 224 us (264), 1.22; 32 experts of
// 0 .. 1100 rows, 1024 x 4096, GELU: 150 us (182), 0.95 (the tiles' rows past the utterances'
// ends not counted); 8 heads of 5 .. 49 rows, 768 x 48: 7.6 us (10.1).
#include <algorithm>

#include "segments.cuh"
#include "w2v_kernels.h"

namespace w2v {
namespace sg {

constexpr int kBM = 128, kBK = 64;
constexpr int kNE = 8;                         // epilogue warps
constexpr int kThreads = 64 + 32 * kNE;
constexpr int kSmemCap = 232448;
constexpr int kABytes = kBM * kBK * 2;
constexpr int kTailBytes = 512;                // barriers, the stages' work
constexpr int kEpiBytes = kNE * 4096;          // per warp: a 32 x 32 fp32 chunk, or two fp16 store boxes
constexpr int kMaxStages = 8;
// A stage's work: its number of MMA steps, these, and a mask from kWrap on: step k takes columns 16 k of
// the rows and 16 (k & mask) of the weights (an adapter's value and remainder meet the same ones).
// kOwned: an adapter's, whose product changes its own rows only.
constexpr uint32_t kLastOfTile = 16, kLastOfSum = 32, kOwned = 64, kWrap = 8, kMainWork = kBK / 16 | (kBK / 16 - 1) << kWrap;
__host__ __device__ constexpr bool sums_of(int epi) { return epi == W2V_EPI_F32 || epi == W2V_EPI_F32_RESID; }
// K-blocks of a sum: 512 of K; beside a residual, which as a rule is larger than what is added to it, 1024.
__host__ __device__ constexpr int sum_blocks(int epi) { return epi == W2V_EPI_F32_RESID ? 16 : 8; }

struct Params {
    int M, N, k_blocks;
    int bn, n_tiles, m_tiles;                  // m_tiles, of rows: lora: all; grouped: no more than so many
    int stages, b_bytes;
    int a_rows;                                // rows of a stage's operand box: 128, lora: fewer where there are no more
    int vec, tma_c, bias_vec, bias_stride;     // wide stores; fp16 tile stores; wide bias loads; grouped: N
    void* C;
    long long ldc;
    const float* bias;
    const float* resid;
    long long ldr;
    int* err;
    // lora
    LoraPlan plan;
    int lora;                                  // the plan holds adapters
    // grouped
    const long long* off;
    const int* T;
    const int* group;
    int n_utt, n_groups;
};

// A tile's rows and weights.
struct Tile {
    int row0, end;                             // first row, one past the last valid row
    int ni, group;
};

// Walks the utterances in steps of 32 (warp-collective): row tile m of the
// batch, for m in ascending order.
struct Walker {
    int base = -32, before = 0;                // utterances base .. base + 31 (one per lane); row tiles before them
    int first = 0, end = 0, group = 0, incl = 0, total = 0;

    W2V_DEV void load(const Params& p, int tile_rows) {
        const int u = base + (int)(threadIdx.x & 31);
        int tiles = 0;
        if (u < p.n_utt) {
            const long long o = p.off[u];
            const int t = p.T[u];
            group = p.group[u];
            if (o >= 0 && o < p.M && t > 0 && group >= 0 && group < p.n_groups) {
                first = (int)o;
                end = (int)min((long long)p.M, o + t);
                tiles = (end - first + tile_rows - 1) / tile_rows;
            }
        }
        incl = tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, d);
            if ((int)(threadIdx.x & 31) >= d) incl += v;
        }
        total = __shfl_sync(0xffffffffu, incl, 31);
    }
    // all row tiles of the batch (utterances that overlap could have more than fit an int)
    W2V_DEV int count(const Params& p, int tile_rows) {
        int n = 0;
        for (base = 0; base < p.n_utt && n < p.m_tiles; base += 32) {
            load(p, tile_rows);
            n = min(n + total, p.m_tiles);
        }
        base = -32;
        total = 0;
        return n;
    }
    // m not below an earlier call's; false: there are no more
    W2V_DEV bool find(const Params& p, int tile_rows, int m, Tile& t) {
        while (m >= before + total) {
            if (base + 32 >= p.n_utt) return false;
            before += total;
            base += 32;
            load(p, tile_rows);
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + incl > m);
        const int src = __ffs(past) - 1;
        const int prev = __shfl_sync(0xffffffffu, incl, src > 0 ? src - 1 : 0);
        const int k = m - before - (src > 0 ? prev : 0);
        t.row0 = uniform(__shfl_sync(0xffffffffu, first, src) + k * tile_rows);
        t.end = uniform(__shfl_sync(0xffffffffu, end, src));
        t.group = uniform(__shfl_sync(0xffffffffu, group, src));
        return true;
    }
};

W2V_DEV float epi_value(int epi, float x) { return epi == W2V_EPI_F16_GELU ? gelu_tanh(x) : x; }

// The residual of this thread's 8 cells (4 columns) of a 32 x 32 chunk.
W2V_DEV void load_resid(const Params& p, int row0, int end, int col0, float4 (&res)[8]) {
    const int lane = threadIdx.x & 31, col = col0 + 4 * (lane & 7);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = row0 + (lane >> 3) + 4 * i;
        res[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r >= end || col >= p.N) continue;
        const float* src = p.resid + (long long)r * p.ldr + col;
        if (p.vec && col + 3 < p.N) res[i] = *reinterpret_cast<const float4*>(src);
        else {
            res[i].x = src[0];
            if (col + 1 < p.N) res[i].y = src[1];
            if (col + 2 < p.N) res[i].z = src[2];
            if (col + 3 < p.N) res[i].w = src[3];
        }
    }
}

// A staged 32 x 32 fp32 chunk to C: 8 threads per row, 4 columns each.
template <int EPI>
W2V_DEV void store_chunk(const Params& p, const float* stg, const float* bias, int row0, int end, int col0,
                         const float4 (&res)[8]) {
    const int lane = threadIdx.x & 31, cg = lane & 7, rs = lane >> 3;
    const int col = col0 + 4 * cg;
    if (col >= p.N) return;
    const int n = min(4, p.N - col);
    float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
    if (bias) {
        if (p.bias_vec && n == 4) b = __ldg(reinterpret_cast<const float4*>(bias + col));
        else {
            b.x = __ldg(bias + col);
            if (n > 1) b.y = __ldg(bias + col + 1);
            if (n > 2) b.z = __ldg(bias + col + 2);
            if (n > 3) b.w = __ldg(bias + col + 3);
        }
    }
    float4 xs[8];
#pragma unroll
    for (int i = 0; i < 8; i++) xs[i] = stage_get(stg, rs + 4 * i, cg);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int r = row0 + rs + 4 * i;
        if (r >= end) continue;
        float4 x = xs[i];
        x.x += b.x; x.y += b.y; x.z += b.z; x.w += b.w;
        if (EPI == W2V_EPI_F32_RESID) { x.x += res[i].x; x.y += res[i].y; x.z += res[i].z; x.w += res[i].w; }
        x.x = epi_value(EPI, x.x); x.y = epi_value(EPI, x.y); x.z = epi_value(EPI, x.z); x.w = epi_value(EPI, x.w);
        const long long at = (long long)r * p.ldc + col;
        if (EPI == W2V_EPI_F16 || EPI == W2V_EPI_F16_GELU) {
            __half* c = reinterpret_cast<__half*>(p.C) + at;
            if (p.vec && n == 4) *reinterpret_cast<uint2*>(c) = make_uint2(pack_half2(x.x, x.y), pack_half2(x.z, x.w));
            else {
                c[0] = __float2half_rn(x.x);
                if (n > 1) c[1] = __float2half_rn(x.y);
                if (n > 2) c[2] = __float2half_rn(x.z);
                if (n > 3) c[3] = __float2half_rn(x.w);
            }
        } else {
            float* c = reinterpret_cast<float*>(p.C) + at;
            if (p.vec && n == 4) *reinterpret_cast<float4*>(c) = x;
            else {
                c[0] = x.x;
                if (n > 1) c[1] = x.y;
                if (n > 2) c[2] = x.z;
                if (n > 3) c[3] = x.w;
            }
        }
    }
}

// One row per lane of an fp16 chunk into a 32-row box of 64-byte rows (64-byte
// swizzle) and out by one TMA tile store, which clips columns past N.
template <int EPI>
W2V_DEV void store_box(const Params& p, const CUtensorMap* tmC, float (&v)[32], const float* bias, uint8_t* box, int row0,
                       int col0) {
    const int lane = threadIdx.x & 31;
    if (bias) {
        if (p.bias_vec && col0 + 32 <= p.N) {
            const float4* b4 = reinterpret_cast<const float4*>(bias + col0);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float4 b = __ldg(b4 + j);
                v[4 * j] += b.x; v[4 * j + 1] += b.y; v[4 * j + 2] += b.z; v[4 * j + 3] += b.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; j++) if (col0 + j < p.N) v[j] += __ldg(bias + col0 + j);
        }
    }
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] = epi_value(EPI, v[j]);
    if (lane == 0) bulk_wait_group_read<1>();      // the store two boxes ago has read this one
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; j++) {
        uint4 u;
        u.x = pack_half2(v[8 * j + 0], v[8 * j + 1]);
        u.y = pack_half2(v[8 * j + 2], v[8 * j + 3]);
        u.z = pack_half2(v[8 * j + 4], v[8 * j + 5]);
        u.w = pack_half2(v[8 * j + 6], v[8 * j + 7]);
        *reinterpret_cast<uint4*>(box + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = u;
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
        tma_store_3d(tmC, box, col0, row0, 0);
        bulk_commit_group();
    }
}

// Two 32 x 32 blocks of TMEM (32 lanes, 32 columns) with one wait.
W2V_DEV void tmem_ld32x2(uint32_t addr_a, float (&a)[32], uint32_t addr_b, float (&b)[32]) {
    uint32_t r[32], s[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%64];\n"
        " tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%65];\n"
        " tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(s[0]), "=r"(s[1]), "=r"(s[2]), "=r"(s[3]), "=r"(s[4]), "=r"(s[5]), "=r"(s[6]), "=r"(s[7]),
          "=r"(s[8]), "=r"(s[9]), "=r"(s[10]), "=r"(s[11]), "=r"(s[12]), "=r"(s[13]), "=r"(s[14]), "=r"(s[15]),
          "=r"(s[16]), "=r"(s[17]), "=r"(s[18]), "=r"(s[19]), "=r"(s[20]), "=r"(s[21]), "=r"(s[22]), "=r"(s[23]),
          "=r"(s[24]), "=r"(s[25]), "=r"(s[26]), "=r"(s[27]), "=r"(s[28]), "=r"(s[29]), "=r"(s[30]), "=r"(s[31])
        : "r"(addr_a), "r"(addr_b)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) { a[i] = __uint_as_float(r[i]); b[i] = __uint_as_float(s[i]); }
}

template <int EPI, bool PAIR, bool LORA>
__global__ void __launch_bounds__(kThreads, 1)
seg_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmT,
                const __grid_constant__ CUtensorMap tmL, const __grid_constant__ Params p) {
    constexpr int CT = PAIR ? 2 : 1, kTileRows = kBM * CT;
    constexpr bool SUMS = sums_of(EPI), WORK = LORA || SUMS;   // WORK: a stage says what is to be done with it
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw);
    // identical offset in both CTAs of a pair: the MMA addresses the peer's operands at the leader's offsets
    uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
    const int S = p.stages, stage_bytes = kABytes + p.b_bytes;
    uint8_t* epi = smem + S * stage_bytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(epi + kEpiBytes);
    uint64_t* empty = full + kMaxStages;
    uint64_t* tfull = empty + kMaxStages;
    uint64_t* tempty = tfull + 2;
    uint64_t* done = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
    uint32_t* stage_work = tmem_slot + 1;      // what the MMA does with a stage
    uint32_t* stage_off = reinterpret_cast<uint32_t*>(epi + kEpiBytes + 256);   // an adapter's: the rows left alone
    static_assert((2 * kMaxStages + 5) * 8 + 4 + 4 * kMaxStages <= 256 && 256 + kMaxStages * kOwnerWords * 4 <= kTailBytes, "tail");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
    const int unit = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
    const int n_units = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

    Walker walk;
    auto tile_at = [&](int tile, Tile& t) {
        t.ni = tile % p.n_tiles;
        const int m = tile / p.n_tiles;
        if constexpr (LORA) { t.row0 = m * kTileRows; t.end = p.M; t.group = 0; return true; }
        else return walk.find(p, kTileRows, m, t);
    };
    Tile tile0 = {};                           // the producer's first, found while the others set up
    bool any = true;
    if (!LORA && warp == 0) any = tile_at(unit, tile0);
    if (threadIdx.x == 32 * (kThreads / 32 - 1)) {
        for (int s = 0; s < S; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; b++) { mbar_init(&tfull[b], 1); mbar_init(&tempty[b], kNE * CT); }
        mbar_init(done, 1);
        fence_mbar_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) {
        if (PAIR) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
        else { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    }
    tc_fence_before();
    if (PAIR) cluster_sync_all(); else __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = (uint32_t)uniform((int)*tmem_slot);

    // accumulators: two, or with running totals (columns 0 .. bn - 1) one or two behind them
    const int n_sums = SUMS ? (p.k_blocks + sum_blocks(EPI) - 1) / sum_blocks(EPI) : 1;
    const uint32_t n_acc = n_sums > 1 && 3 * p.bn > 512 ? 1u : 2u;
    auto accumulator_at = [&](uint32_t i) {
        return tmem_base + (n_sums > 1 ? (uint32_t)p.bn * (1u + i) : i * 256u);
    };
    // the producer walks until there are no more tiles; the others count them while it loads the first
    const int total = (LORA || warp == 0 ? p.m_tiles : walk.count(p, kTileRows)) * p.n_tiles;
    // further K-blocks of a row tile: adapters x groups of 32 ranks
    const int chunks = LORA ? (p.plan.rank + kGroup - 1) / kGroup : 0;

    if (warp == 0) {
        // the leader's barriers count the bytes of a pair
        const uint32_t lead = elect_one(), full_lead = PAIR ? mapa_shared(smem_u32(full), 0) : smem_u32(full);
        const uint32_t arm = lead & (uint32_t)(rank == 0), base = smem_u32(smem);
        uint32_t arm_bytes = 0;                // of a stage, both CTAs' in a pair
        const int b_row = (int)rank * (p.bn / 2);
        int stage = 0;
        uint32_t phase = 0, issued = 0, last_par = 0;
        bool ok = true;
        // one stage's two tiles; work: its MMA steps, and whether it is the last of a sum and of the tile
        // grouped: of the rows only the 32-row boxes that hold valid ones, where that saves any (tmT, which is
        // theirs then): what the MMA reads in the others' places goes to accumulator rows that are not stored
        int boxes = 4;
        // owners of four of the tile's blocks, a word per lane, and which of the four the stage's is
        uint32_t owners = 0;
        int owner_at = 0;
        // k, kw: first column of the rows' and of the weights' tile
        auto stage_in = [&](const CUtensorMap* ma, const CUtensorMap* mb, int k, int ra, int rb, int gb, uint32_t work, int kw) {
            if (!mbar_wait_warp(&empty[stage], phase ^ 1u, p.err)) { ok = false; return; }
            const uint32_t dst = base + (uint32_t)(stage * stage_bytes), bar = full_lead + (uint32_t)(stage * 8);
            if (WORK && lane == 0) stage_work[stage] = work;
            const bool owned = LORA && (work & kOwned);
            if (WORK && !owned) __syncwarp();
            if (!owned) expect_tx_if(arm, smem_u32(&full[stage]), arm_bytes);
            if (LORA || boxes == 4) {
                tma_load_2d_if<PAIR>(lead, dst, ma, bar, k, ra + (int)rank * kBM);
            } else {
                for (int i = 0; i < boxes; i++)
                    tma_load_2d_if<PAIR>(lead, dst + (uint32_t)(i * kABytes / 4), &tmT, bar, k, ra + (int)rank * kBM + i * 32);
            }
            tma_load_3d_if<PAIR>(lead, dst + kABytes, mb, bar, kw, rb + b_row, gb);
            if (owned) {                       // (behind the loads: the owners may still be on their way)
                if (lane / kOwnerWords == owner_at) stage_off[stage * kOwnerWords + lane % kOwnerWords] = ~owners;
                __syncwarp();
                expect_tx_if(arm, smem_u32(&full[stage]), arm_bytes);
            }
            issued |= 1u << stage;
            last_par = (last_par & ~(1u << stage)) | (phase << stage);
            if (++stage == S) { stage = 0; phase ^= 1u; }
        };
        for (int tile = unit; tile < total && any && ok; tile += n_units) {
            Tile t = tile0;
            if ((LORA || tile != unit) && !tile_at(tile, t)) break;
            const int col0 = t.ni * p.bn;
            if constexpr (LORA) {
                arm_bytes = (uint32_t)(CT * (p.b_bytes + p.a_rows * kBK * 2));
            } else {
                auto boxes_of = [&](int r) { return max(min((t.end - r + 31) / 32, 4), 0); };
                boxes = boxes_of(t.row0 + (int)rank * kBM);
                arm_bytes = (uint32_t)(CT * p.b_bytes + (boxes_of(t.row0) + (PAIR ? boxes_of(t.row0 + kBM) : 0)) * (kABytes / 4));
            }
            for (int kb = 0; kb < p.k_blocks - 1 && ok; kb++)
                stage_in(&tmA, &tmB, kb * kBK, t.row0, col0, t.group,
                         kMainWork | (SUMS && kb % sum_blocks(EPI) == sum_blocks(EPI) - 1 ? kLastOfSum : 0), kb * kBK);
            int blocks = 0, first = 0, rec = 0;
            if (LORA && p.lora) {
                if (tile == unit) grid_dependency_wait();
                // the tile's record: first block, their number, the adapters of the first ones
                rec = lane < 2 + kInline ? reinterpret_cast<const int*>(p.plan.tiles + t.row0 / kTileRows)[lane] : 0;
                first = uniform(__shfl_sync(0xffffffffu, rec, 0));
                blocks = uniform(__shfl_sync(0xffffffffu, rec, 1));
            }
            auto owners_from = [&](int b) {
                if (b + lane / kOwnerWords < blocks) owners = p.plan.owners[(long long)(first + b) * kOwnerWords + lane];
            };
            owners_from(0);
            if (ok)
                stage_in(&tmA, &tmB, (p.k_blocks - 1) * kBK, t.row0, col0, t.group, kMainWork | (blocks ? 0 : kLastOfTile | kLastOfSum), (p.k_blocks - 1) * kBK);
            for (int b = 0; b < blocks && ok; b++) {
                const int held = __shfl_sync(0xffffffffu, rec, min(2 + b, 31));
                const int ad = uniform(b < kInline ? held : p.plan.adapter[first + b]);
                owner_at = b % (32 / kOwnerWords);
                if (b && owner_at == 0) owners_from(b);
                for (int c = 0; c < chunks && ok; c++) {
                    const uint32_t steps = (uint32_t)group_width(p.plan.rank, c * kGroup) / 16;
                    const bool last = b + 1 == blocks && c + 1 == chunks;
                    stage_in(&tmT, &tmL, c * kBK, (first + b) * kTileRows, col0, ad,
                             kOwned | 2 * steps | (steps - 1) << kWrap | (last ? kLastOfTile | kLastOfSum : 0), c * kGroup);
                }
            }
        }
        // no bulk copy may still be writing shared memory when the CTA (or its peer) exits
        if (lane == 0 && rank == 0)
            for (int s = 0; s < S; s++)
                if (issued & (1u << s)) mbar_wait(&full[s], (last_par >> s) & 1u, p.err);
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = umma_idesc_f16(kTileRows, p.bn), lead = elect_one();
            const uint64_t desc0 = umma_desc_sw128(smem_u32(smem));
            const uint32_t empty_here = smem_u32(empty), empty_peer = PAIR ? mapa_shared(smem_u32(empty), 1) : 0u;
            const uint32_t tfull_here = smem_u32(tfull), tfull_peer = PAIR ? mapa_shared(smem_u32(tfull), 1) : 0u;
            int stage = 0;
            uint32_t phase = 0, acc = 0, acc_phase = 0;
            bool ok = true;
            for (int tile = unit; tile < total && ok; tile += n_units) {
                bool first = true;               // stage of a sum
                uint32_t d = 0;
                // a stage's operands are there, and an accumulator for the first of a sum
                auto begin = [&] {
                    if (first) {
                        if (!mbar_wait_warp(&tempty[acc], acc_phase ^ 1u, p.err)) return false;
                        d = accumulator_at(acc);
                    }
                    if (!mbar_wait_warp(&full[stage], phase, p.err)) return false;
                    tc_fence_after();
                    return true;
                };
                auto multiply = [&](uint32_t go, int kk) {
                    const uint64_t da = desc_plus(desc0, (uint32_t)(stage * stage_bytes)), db = desc_plus(da, kABytes);
                    umma_f16_if<PAIR>(go, d, desc_plus(da, kk * 32), desc_plus(db, kk * 32), idesc, !first || kk != 0);
                };
                auto end = [&](bool last_of_sum) {
                    umma_commit_if<PAIR>(lead, empty_here + (uint32_t)(stage * 8));
                    if (PAIR) umma_commit_if<PAIR>(lead, empty_peer + (uint32_t)(stage * 8));
                    if (++stage == S) { stage = 0; phase ^= 1u; }
                    first = last_of_sum;
                    if (last_of_sum) {
                        umma_commit_if<PAIR>(lead, tfull_here + acc * 8u);
                        if (PAIR) umma_commit_if<PAIR>(lead, tfull_peer + acc * 8u);
                        if (++acc == n_acc) { acc = 0; acc_phase ^= 1u; }
                    }
                };
                // (a loop for these alone: with the adapters' stages in it, each a look at its work and MMAs
                // under its predicate, 64 x 10 s of 768 x 2304 took 112 us, not 104, 31 K rows of 1024 x 4096 246, not 221)
                for (int kb = 0; kb < p.k_blocks - 1; kb++) {
                    if (!begin()) { ok = false; break; }
#pragma unroll
                    for (int kk = 0; kk < kBK / 16; kk++) multiply(lead, kk);
                    end(SUMS && kb % sum_blocks(EPI) == sum_blocks(EPI) - 1);
                }
                // the last of K and the adapters' stages: as the producer found them
                for (uint32_t work = 0; ok && !(work & kLastOfTile);) {
                    if (!begin()) { ok = false; break; }
                    work = WORK ? (uint32_t)uniform((int)stage_work[stage]) : kMainWork | kLastOfSum | kLastOfTile;
                    if (LORA && (work & kOwned)) {
                        const uint4* words = reinterpret_cast<const uint4*>(stage_off + stage * kOwnerWords);
                        const uint4 o0 = words[0], o1 = words[PAIR ? 1 : 0];
                        const uint32_t off[kOwnerWords] = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, o1.z, o1.w};
                        const uint64_t da = desc_plus(desc0, (uint32_t)(stage * stage_bytes)), db = desc_plus(da, kABytes);
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; kk++)
                            umma_f16_masked_if<PAIR>(lead & (uint32_t)(kk < (int)(work & 15u)), d, desc_plus(da, kk * 32),
                                                     desc_plus(db, (kk & (int)(work >> kWrap)) * 32), idesc, off);
                    } else {
#pragma unroll
                        for (int kk = 0; kk < kBK / 16; kk++) multiply(lead, kk);
                    }
                    end((work & kLastOfSum) != 0);
                }
            }
            // no MMA may still be writing TMEM when it is freed (also after an expired wait)
            umma_commit_if<PAIR>(lead, smem_u32(done));
            mbar_wait(done, 0, p.err);
        }
        __syncwarp();
    } else {
        const int q = warp & 3;                 // TMEM lane quarter this warp may access
        const int n_ch = p.bn / 32, half = (n_ch + 1) / 2;
        const int c0 = warp < 6 ? 0 : half, c1 = warp < 6 ? half : n_ch;   // two warps per quarter
        const uint32_t tempty_lead = PAIR ? mapa_shared(smem_u32(tempty), 0) : 0u;
        float* stg = reinterpret_cast<float*>(epi + (warp - 2) * 4096);
        constexpr bool kF16 = EPI == W2V_EPI_F16 || EPI == W2V_EPI_F16_GELU;
        uint32_t nst = 0, acc = 0, acc_phase = 0;
        for (int tile = unit; tile < total; tile += n_units) {
            Tile t;
            tile_at(tile, t);
            const int row0 = t.row0 + (int)rank * kBM + q * 32;
            const int col0 = t.ni * p.bn;
            const float* bias = p.bias ? p.bias + (long long)t.group * p.bias_stride : nullptr;
            // whole boxes inside the rows to be written (lora: the map clips at M)
            const bool box = kF16 && p.tma_c && (LORA ? row0 < t.end : row0 + 32 <= t.end);
            const uint32_t lanes = (uint32_t)(q * 32) << 16;
            auto release = [&]() {               // hands the accumulator back
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) mbar_arrive_remote(tempty_lead + acc * 8u);
                    else mbar_arrive(&tempty[acc]);
                }
                if (++acc == n_acc) { acc = 0; acc_phase ^= 1u; }
            };
            float4 res[8];
            if (EPI == W2V_EPI_F32_RESID && c0 < c1) load_resid(p, row0, t.end, col0 + c0 * 32, res);
            uint32_t from = tmem_base;           // where the finished sums are
            bool ok = true;
            for (int s = 0; s < n_sums; s++) {
                if (!mbar_wait_warp(&tfull[acc], acc_phase, p.err)) { ok = false; break; }
                tc_fence_after();
                if (n_sums == 1) {
                    from = accumulator_at(acc);
                } else {
#pragma unroll 1
                    for (int c = c0; c < c1; c++) {
                        float v[32], w[32];
                        const uint32_t sum = tmem_base + lanes + (uint32_t)(c * 32);
                        tmem_ld32x2(accumulator_at(acc) + lanes + (uint32_t)(c * 32), v, sum, w);
#pragma unroll
                        for (int j = 0; j < 32; j++) v[j] = s ? v[j] + w[j] : v[j];
                        tmem_st32(sum, v);
                    }
                    release();
                }
            }
            if (!ok) break;
            if (kF16 && !box && nst) {           // boxes become the staging buffer
                if (lane == 0) bulk_wait_group_read<0>();
                __syncwarp();
            }
            if (row0 < t.end) {
#pragma unroll 1
                for (int c = c0; c < c1; c++) {
                    const int cc = col0 + c * 32;
                    if (cc >= p.N) break;
                    float v[32];
                    tmem_ld32(from + lanes + (uint32_t)(c * 32), v);
                    if (kF16 && box) {
                        store_box<EPI>(p, &tmC, v, bias, reinterpret_cast<uint8_t*>(stg) + (nst & 1u) * 2048, row0, cc);
                        nst++;
                        continue;
                    }
                    float4 cur[8];
                    if (EPI == W2V_EPI_F32_RESID) {
#pragma unroll
                        for (int i = 0; i < 8; i++) cur[i] = res[i];
                        // the next chunk's residual is in flight while this chunk is stored
                        if (c + 1 < c1) load_resid(p, row0, t.end, cc + 32, res);
                    }
                    __syncwarp();
                    stage_put(stg, v);
                    __syncwarp();
                    store_chunk<EPI>(p, stg, bias, row0, t.end, cc, cur);
                }
                __syncwarp();
            }
            if (n_sums == 1) release();
        }
        if (kF16) {      // the stores are complete before the CTA exits
            if (lane == 0) bulk_wait_group<0>();
            __syncwarp();
        }
    }

    tc_fence_before();
    if (PAIR) cluster_sync_all(); else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        if (PAIR) tmem_dealloc_pair(tmem_base, 512); else tmem_dealloc(tmem_base, 512);
    }
}

// ── host side ───────────────────────────────────────────────────────────────

struct Maps {
    CUtensorMap a, b, c, t, l;
};

template <int EPI, bool PAIR, bool LORA>
static int launch(const Maps& m, const Params& p, int tiles, bool dependent, cudaStream_t st) {
    auto kern = seg_gemm_kernel<EPI, PAIR, LORA>;
    static int max_units[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (PAIR) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 2;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = kSmemCap;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    if (!max_units[dev & 63]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemCap) != cudaSuccess)
            return W2V_ERR_LAUNCH;
        int sms = 0;
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 2) return W2V_ERR_LAUNCH;
        int units = sms / (PAIR ? 2 : 1);
        if (PAIR) {          // pairs that can be resident at once (a GPC may leave an SM unpaired)
            cfg.gridDim = dim3(2 * (sms / 2), 1, 1);
            int c = 0;
            if (cudaOccupancyMaxActiveClusters(&c, kern, &cfg) == cudaSuccess && c > 0) units = c;
            cudaGetLastError();
        }
        max_units[dev & 63] = units;
    }
    const int units = tiles < max_units[dev & 63] ? tiles : max_units[dev & 63];
    cfg.gridDim = dim3((unsigned)(units * (PAIR ? 2 : 1)), 1, 1);
    if (dependent) {         // start while the first product runs
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = ++n;
    }
    if (cudaLaunchKernelEx(&cfg, kern, m.a, m.b, m.c, m.t, m.l, p) != cudaSuccess) return W2V_ERR_LAUNCH;
    return cudaPeekAtLastError() == cudaSuccess ? W2V_OK : W2V_ERR_LAUNCH;
}

template <bool PAIR, bool LORA>
static int launch_epi(int epi, const Maps& m, const Params& p, int tiles, bool dependent, cudaStream_t st) {
    switch (epi) {
        case W2V_EPI_F16: return launch<W2V_EPI_F16, PAIR, LORA>(m, p, tiles, dependent, st);
        case W2V_EPI_F16_GELU: return launch<W2V_EPI_F16_GELU, PAIR, LORA>(m, p, tiles, dependent, st);
        case W2V_EPI_F32: return launch<W2V_EPI_F32, PAIR, LORA>(m, p, tiles, dependent, st);
        default: return launch<W2V_EPI_F32_RESID, PAIR, LORA>(m, p, tiles, dependent, st);
    }
}

// Tile: width w (a multiple of 32) and single CTAs or pairs, by waves over the
// SMs x the cycles of a tile.  A K-block of 64 takes an SM 2 w cycles of MMA; its
// operands, 16 KB of rows and 128 w bytes of weights (half of that in a pair, which
// shares them), are counted at 64 bytes a cycle (a model, which orders the widths: the
// path itself takes about twice as much).  A wave also has a fill, a drain and an epilogue.
static void pick_tile(int N, long long m_tiles1, long long m_tiles2, long long K, int* bn, bool* pair) {
    double best = 1e300;
    for (int pr = 0; pr < 2; pr++)
        for (int w = 32; w <= 256; w += 32) {
            if (w > 32 && w - 32 >= N) continue;
            const long long tiles = (pr ? m_tiles2 : m_tiles1) * ((N + w - 1) / w);
            const long long slots = pr ? 74 : 148;
            const long long waves = (tiles + slots - 1) / slots;
            const double block = std::max(2.0 * w, 256.0 + (pr ? 1.0 : 2.0) * w);
            const double cost = (double)waves * (K / kBK * block + 600 + 6.0 * w);
            if (cost < best) { best = cost; *bn = w; *pair = pr != 0; }
        }
}

struct Call {
    const void* A;
    long long lda, K, M;
    const void* B;
    int n_mats, N;             // weight matrices (1: shared)
    void* C;
    long long ldc;
    const float* bias;
    const float* resid;
    long long ldr;
    int epilogue;
    const long long* off;
    const int* T;
    const int* index;
    int n_utt;
    int* err;
};

static bool refused(const Call& c) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(c.A), b = reinterpret_cast<uintptr_t>(c.B);
    if (c.K <= 0 || c.K % 64 || c.K > 0x7fffffffLL || c.M < 0 || c.M > 0x7fffffffLL - 512 || c.N <= 0 || c.N > 0x7fffffff - 512 ||
        c.n_utt > 0x7fffffff - 512 || c.lda < c.K || c.lda % 8 || c.ldc < c.N || ((a | b) & 15) || c.epilogue < W2V_EPI_F16 || c.epilogue > W2V_EPI_F32_RESID ||
        c.n_utt < 0)
        return true;
    return c.M > 0 && (!c.A || !c.B || !c.C || (c.epilogue == W2V_EPI_F32_RESID && (!c.resid || c.ldr < c.N)) ||
                       (c.n_utt > 0 && (!c.off || !c.T || !c.index)));
}

// Parameters and maps that both products share.
static int common(const Call& c, bool lora, int bn, bool pair, Params& p, Maps& m) {
    const bool f16 = c.epilogue == W2V_EPI_F16 || c.epilogue == W2V_EPI_F16_GELU;
    const uintptr_t C = reinterpret_cast<uintptr_t>(c.C), R = reinterpret_cast<uintptr_t>(c.resid);
    p.M = (int)c.M;
    p.N = c.N;
    p.k_blocks = (int)(c.K / kBK);
    p.bn = bn;
    p.n_tiles = (c.N + bn - 1) / bn;
    p.b_bytes = (pair ? bn / 2 : bn) * kBK * 2;
    p.stages = std::min(kMaxStages, (kSmemCap - 1024 - kTailBytes - kEpiBytes) / (kABytes + p.b_bytes));
    p.vec = c.ldc % 4 == 0 && C % (f16 ? 8 : 16) == 0 &&
            (c.epilogue != W2V_EPI_F32_RESID || (c.ldr % 4 == 0 && R % 16 == 0));
    p.bias_vec = reinterpret_cast<uintptr_t>(c.bias) % 16 == 0 && (c.n_mats == 1 || c.N % 4 == 0);
    p.bias_stride = c.n_mats == 1 ? 0 : c.N;
    p.C = c.C;
    p.ldc = c.ldc;
    p.bias = c.bias;
    p.resid = c.resid;
    p.ldr = c.ldr;
    p.err = c.err;
    const uint64_t ad[2] = {(uint64_t)c.K, (uint64_t)c.M}, as[1] = {(uint64_t)c.lda * 2};
    p.a_rows = lora && c.M < kBM ? (int)((c.M + 31) / 32 * 32) : kBM;
    int rc = map_f16(&m.a, c.A, 2, ad, as, p.a_rows);
    if (rc) return rc;
    m.c = m.t = m.l = m.a;
    if (!lora) rc = map_f16(&m.t, c.A, 2, ad, as, 32);
    if (rc) return rc;
    const uint64_t bd[3] = {(uint64_t)c.K, (uint64_t)c.N, (uint64_t)c.n_mats};
    const uint64_t bs[2] = {(uint64_t)c.K * 2, (uint64_t)c.K * 2 * c.N};
    rc = map_f16(&m.b, c.B, 3, bd, bs, pair ? bn / 2 : bn);
    if (rc) return rc;
    // fp16 C by 32 x 32 boxes; a store clips the innermost dimension at 16-byte granularity only
    p.tma_c = f16 && c.ldc % 8 == 0 && c.N % 8 == 0 && C % 16 == 0;
    if (p.tma_c) {
        const uint64_t cd[3] = {(uint64_t)c.N, (uint64_t)c.M, 1};
        const uint64_t cs[2] = {(uint64_t)c.ldc * 2, (uint64_t)c.ldc * 2 * c.M};
        const uint32_t cbox[3] = {32, 32, 1}, es[3] = {1, 1, 1};
        if (get_encode()(&m.c, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, c.C, cd, cs, cbox, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return W2V_ERR_TENSOR_MAP;
    }
    return W2V_OK;
}

}  // namespace sg
}  // namespace w2v

using namespace w2v::sg;

extern "C" long long w2v_lora_workspace_bytes(long long M, int n_utt, int rank) {
    if (M < 0 || M > 0x7fffffffLL - 512 || n_utt < 0 || n_utt > 0x7fffffff - 512 || rank < 8 || rank > 128 || rank % 8) return -1;
    return lora_workspace(M, n_utt, rank);
}

extern "C" int w2v_gemm_f16_lora(const void* A, long long lda, long long K, long long M, const void* B, int N, void* C,
                                 long long ldc, const float* bias, const float* resid, long long ldr, int epilogue,
                                 const void* lora_a, const void* lora_b, const float* lora_scale, int n_adapters,
                                 int rank, const long long* off, const int* T, const int* adapter, int n_utt,
                                 void* workspace, long long workspace_bytes, int* err, void* stream) {
    const Call c{A, lda, K, M, B, 1, N, C, ldc, bias, resid, ldr, epilogue, off, T, adapter, n_utt, err};
    if (refused(c) || !B || rank < 8 || rank > 128 || rank % 8 || n_adapters <= 0 || !lora_a || !lora_b ||
        ((reinterpret_cast<uintptr_t>(lora_a) | reinterpret_cast<uintptr_t>(lora_b)) & 15))
        return W2V_ERR_ARGS;
    if (M == 0) return W2V_OK;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 127)) return W2V_ERR_ARGS;
    const long long need = lora_workspace(M, n_utt, rank);
    if (need < 0) return W2V_ERR_ARGS;
    if (workspace_bytes < need) return W2V_ERR_CAPACITY;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    Params p = {};
    Maps m;
    int bn = 256;
    bool pair = false;
    pick_tile(N, (M + 127) / 128, (M + 255) / 256, K, &bn, &pair);
    int rc = common(c, true, bn, pair, p, m);
    if (rc) return rc;
    const int tile_rows = pair ? 256 : 128;
    p.m_tiles = (int)((M + tile_rows - 1) / tile_rows);
    p.lora = n_utt > 0;
    p.plan = lora_plan(workspace, M, n_utt, rank, tile_rows);
    if (p.lora) {
        const uint64_t td[2] = {(uint64_t)t_columns(rank), (uint64_t)(p.plan.blocks * tile_rows)};
        const uint64_t ts[1] = {(uint64_t)t_columns(rank) * 2};
        rc = map_f16(&m.t, p.plan.t, 2, td, ts, p.a_rows);
        if (rc) return rc;
        const uint64_t ld[3] = {(uint64_t)rank, (uint64_t)N, (uint64_t)n_adapters};
        const uint64_t ls[2] = {(uint64_t)rank * 2, (uint64_t)rank * 2 * N};
        rc = map_f16(&m.l, lora_b, 3, ld, ls, pair ? bn / 2 : bn);
        if (rc) return rc;
        LoraArgs a;
        a.x = reinterpret_cast<const __half*>(A);
        a.lda = lda;
        a.K = (int)K;
        a.M = M;
        a.a = reinterpret_cast<const __half*>(lora_a);
        a.scale = lora_scale;
        a.n_adapters = n_adapters;
        a.off = off;
        a.T = T;
        a.adapter = adapter;
        a.n_utt = n_utt;
        a.err = err;
        a.sums = sums_of(epilogue);
        rc = lora_shrink(a, p.plan, &m.a, p.a_rows, st);
        if (rc) return rc;
    }
    const long long tiles = (long long)p.m_tiles * p.n_tiles;
    if (tiles > 0x7fffffffLL / 2) return W2V_ERR_ARGS;
    return pair ? launch_epi<true, true>(epilogue, m, p, (int)tiles, p.lora, st)
                : launch_epi<false, true>(epilogue, m, p, (int)tiles, p.lora, st);
}

extern "C" int w2v_gemm_grouped_f16(const void* A, long long lda, long long K, long long M, const void* B,
                                    int n_groups, int N, void* C, long long ldc, const float* bias,
                                    const float* resid, long long ldr, int epilogue, const long long* off,
                                    const int* T, const int* group, int n_utt, int* err, void* stream) {
    const Call c{A, lda, K, M, B, n_groups, N, C, ldc, bias, resid, ldr, epilogue, off, T, group, n_utt, err};
    if (n_groups <= 0 || refused(c)) return W2V_ERR_ARGS;
    if (M == 0 || n_utt == 0) return W2V_OK;
    Params p = {};
    Maps m;
    int bn = 256;
    bool pair = false;
    // row tiles: as if the rows were spread evenly, and (below) at most one more than its rows
    // need per utterance
    const long long more = n_utt < M ? n_utt : M, mean = M / more;
    pick_tile(N, more * ((mean + 127) / 128), more * ((mean + 255) / 256), K, &bn, &pair);
    int rc = common(c, false, bn, pair, p, m);
    if (rc) return rc;
    p.off = off;
    p.T = T;
    p.group = group;
    p.n_utt = n_utt;
    p.n_groups = n_groups;
    const long long m_tiles = M / (pair ? 256 : 128) + more, tiles = m_tiles * p.n_tiles;
    if (tiles > 0x7fffffffLL / 2) return W2V_ERR_ARGS;
    p.m_tiles = (int)m_tiles;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return pair ? launch_epi<true, false>(epilogue, m, p, (int)tiles, false, st)
                : launch_epi<false, false>(epilogue, m, p, (int)tiles, false, st);
}
