// First product of the low-rank adapters: t = s_a A_a x for every row, written
// as the masked fp16 blocks that the projections add as further K-blocks
// (segments.cuh).
//
// 2 M K rank operations on M K fp16 values: with the ranks in use (8 .. 128)
// the read of x bounds it, and the time from a block's start to its end where
// there are few rows.  A block takes 128 rows, or 64 where those are few or the
// row tile is no multiple of 128 (the MMA's other 64 rows are then whatever lies
// behind them).  Nine warps: four look up the block's adapters (the plan) and write
// the results, one fills a ring of stages of 64 columns of x and of A_a by TMA, x
// at once and A_a when the plan is there, and up to four multiply.  A stage meets
// each of two adapters, if the rows use two, in accumulators side by side in TMEM,
// so that a block that sees the end of an utterance takes hardly longer than the
// others; more are taken in turn, by other blocks where there are few rows.
// (With m16n8k16 MMAs in registers their rate was the bound: 60 x 10 s, K 1024,
// rank 64 took 31 us.)
//
// Four issuing warps: a stage's wait, MMAs and commit cost one warp some 500 cycles
// where the tensor core takes 184 (four MMAs of 16 columns), a stage after the other.
// Each takes every fourth stage into accumulators of its own, which are added when
// they are read.
//
// Sums over K: for fp32 outputs an issuer's end every 512 of its K, as the projection's do
// (segment_gemm.cu says why); the planning warps then add them to totals with columns of their own,
// and the issuers wait until that is done.  Up to K = 2048 (rank 32 and below) there is one sum.
//
// Few rows (kDirect): what counts is the way from the launch to the results.
// Each adapter has a block of its own whether the rows use it or not, which loads and
// multiplies before the plan is there.  Projections with adapters, the whole call from a short
// graph: 16 single frames of 8 adapters, K = N = 1024, 13.2 us (one warp, and the plan first:
// 1.9 more); 499 rows, K = N = 768, 4 adapters 10.3 (1.7 more).  Call after call the host's issue
// of the two launches is more than that, 15.7 and 14.4 us.
#include "segments.cuh"
#include "w2v_kernels.h"

namespace w2v {
namespace sg {

constexpr int kStep = 64, kMaxTile = 256;
constexpr int kPlanners = 128, kProducer = kPlanners / 32, kIssuers = 4, kThreads = kPlanners + 32 + 32 * kIssuers;
constexpr int kMaxRing = 8;
constexpr int kSumSteps = 512 / kStep;         // K-steps of a sum
// Blocks up to which each adapter has its own: up to 32 the call gains 0.6 to 1.8 us (of 10 to 24);
// at 64 some gain 0.2 to 1.0, others lose 1.9 to 2.5, the blocks standing where the projection's would start.
constexpr int kDirect = 32;

struct ShrinkShape {
    int stages, stage_bytes, smem, cols;       // cols: of TMEM
    int issuers;                               // warps that multiply
    int sums;                                  // of an issuer's over K
    int direct;                                // block y takes adapter y, used or not
    int x_bytes;                               // of a box of x
};
// Two blocks per SM where a ring of three stages or more allows it.
static ShrinkShape shrink_shape(int rows, int rank, int k_steps, bool sums) {
    ShrinkShape s;
    s.stage_bytes = (rows + 2 * rank) * kStep * 2;
    const int behind = 64 * kStep * 2 + 1024;  // what the last stage's MMAs may read past it
    const int two = (108 * 1024 - behind) / s.stage_bytes, one = (216 * 1024 - behind) / s.stage_bytes;
    s.stages = two >= 3 ? two : one;
    if (s.stages > kMaxRing) s.stages = kMaxRing;
    if (s.stages > 3) s.stages &= ~1;
    s.smem = 1024 + s.stages * s.stage_bytes + behind + 256;
    const int acc = 2 * ((rank + 15) / 16 * 16);
    s.issuers = kIssuers;
    auto n_sums = [&] { return sums ? (k_steps + kSumSteps * s.issuers - 1) / (kSumSteps * s.issuers) : 1; };
    auto columns = [&] { return (s.issuers + (n_sums() > 1 ? 1 : 0)) * acc; };
    while (s.issuers > 1 && (columns() > 256 || s.stages % s.issuers)) s.issuers /= 2;
    s.sums = n_sums();
    s.cols = 32;
    while (s.cols < columns()) s.cols *= 2;    // (at most 256 and the totals' 256)
    return s;
}

// 16 columns of TMEM of this warp's lanes <- 16 registers.
W2V_DEV void tmem_st16(uint32_t taddr, const float (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
        "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
        "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
        "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15]))
        : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Barriers of the four warps that plan.
W2V_DEV void plan_sync() { asm volatile("barrier.sync 1, 128;" ::: "memory"); }
W2V_DEV int plan_count(bool x) {
    int n;
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.s32 p, %1, 0;\n barrier.red.popc.u32 %0, 1, 128, p;\n}"
        : "=r"(n)
        : "r"((int)x)
        : "memory");
    return n;
}

template <int kRows>
__global__ void __launch_bounds__(kThreads)
lora_shrink_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, LoraArgs a, LoraPlan p,
                   ShrinkShape shape) {
    constexpr int kXBytes = kRows * kStep * 2;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint16_t seg_start[kMaxTile], seg_end[kMaxTile];   // the tile's utterances that have rows in it
    __shared__ __align__(16) int seg_adapter[kMaxTile];
    __shared__ int16_t seg_slot[kMaxTile];
    __shared__ int slots[kMaxTile];           // the tile's adapters, by their first row
    __shared__ int16_t here[kMaxTile];        // those of them that this block's rows use, then the others
    __shared__ uint8_t present[kMaxTile];
    __shared__ uint32_t present_mask;
    __shared__ int counts[kPlanners / 32];
    __shared__ int row_slot[128];             // of this block's rows
    __shared__ int n_here_shared;
    __shared__ uint64_t full[kMaxRing], empty[kMaxRing], done, drained;
    __shared__ uint32_t tmem_slot;
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* ring = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    const int S = shape.stages;
    const int rank = p.rank, n16 = rank16(rank), a_bytes = rank * kStep * 2;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const long long row0 = (long long)blockIdx.x * kRows;
    const long long tile = row0 / p.tile;
    const long long tile0 = tile * p.tile;
    const int n_rows = (int)min((long long)p.tile, a.M - tile0);
    const int local0 = (int)(row0 - tile0);
    const int k_steps = a.K / kStep;
    const bool direct = shape.direct != 0;
    // the block that is sure to use its rows fetches the first of them before it knows the adapters
    const int early = blockIdx.y == 0 && !direct ? min(S, k_steps) : 0;
    const int issuers = shape.issuers, acc_cols = 2 * n16, sums = shape.sums;
    const int sum_steps = sums > 1 ? kSumSteps * issuers : k_steps;       // of all issuers

    // a stage's x and the adapters' share complete on full[st]
    const uint32_t ring0 = smem_u32(ring), full0 = smem_u32(full), lead = elect_one();
    auto load_x = [&](int st, int ks) {
        tma_load_2d_if<false>(lead, ring0 + (uint32_t)(st * shape.stage_bytes), &tmX, full0 + (uint32_t)(st * 8), ks * kStep,
                              (int)row0);
    };
    int st = 0, used = 0;                     // the producer's: its stage, and stages filled so far
    uint32_t odd = 0, issued = 0;
    bool ok = true;
    auto fill = [&](int n, int ad0, int ad1) {        // x and n adapters' A
        for (int ks = 0; ks < k_steps; ks++) {
            if (used >= S && !mbar_wait_warp(&empty[st], odd ^ 1u, a.err)) { ok = false; break; }
            const uint32_t sa = ring0 + (uint32_t)(st * shape.stage_bytes + kXBytes), bar = full0 + (uint32_t)(st * 8);
            expect_tx_if(lead, bar, (uint32_t)(n * a_bytes + (used >= early ? shape.x_bytes : 0)));
            tma_load_3d_if<false>(lead, sa, &tmA, bar, ks * kStep, 0, ad0);
            if (n > 1) tma_load_3d_if<false>(lead, sa + (uint32_t)a_bytes, &tmA, bar, ks * kStep, 0, ad1);
            if (used >= early) load_x(st, ks);
            issued |= 1u << st;
            used++;
            if (++st == S) { st = 0; odd ^= 1u; }
        }
    };
    // K-steps w, w + issuers, .. of a pass into issuer w's own accumulators; the pass begins at stage `st`.
    // The ring is a multiple of the issuers, so that a stage is always the same one's: another could look
    // for its second filling while the first is on its way, and take the phase before for it.
    auto multiply = [&](int n, int pass) {
        const int w = warp - kProducer - 1;
        if (w >= issuers) return;
        const uint32_t idesc = umma_idesc_f16(128, n16), d0 = (uint32_t)uniform((int)tmem_slot) + (uint32_t)(w * acc_cols);
        const uint64_t desc0 = umma_desc_sw128(smem_u32(ring));
        int at = st + w;
        uint32_t par = odd;
        if (at >= S) { at -= S; par ^= 1u; }
        for (int ks0 = 0, sum = pass * sums; ks0 < k_steps; ks0 += sum_steps, sum++) {
            if (sum > 0 && ok && !mbar_wait_warp(&drained, (uint32_t)(sum - 1) & 1u, a.err)) ok = false;
            tc_fence_after();
            for (int ks = ks0 + w; ks < min(ks0 + sum_steps, k_steps) && ok; ks += issuers) {
                if (!mbar_wait_warp(&full[at], par, a.err)) { ok = false; break; }
                tc_fence_after();
                const uint64_t dx = desc_plus(desc0, (uint32_t)(at * shape.stage_bytes));
                for (int e = 0; e < n; e++) {
                    const uint64_t db = desc_plus(dx, (uint32_t)(kXBytes + e * a_bytes));
                    const uint32_t d = d0 + (uint32_t)(e * n16);
#pragma unroll
                    for (int kk = 0; kk < kStep / 16; kk++)
                        umma_f16_if<false>(lead, d, desc_plus(dx, kk * 32), desc_plus(db, kk * 32), idesc, ks != ks0 + w || kk != 0);
                }
                umma_commit_if<false>(lead, smem_u32(&empty[at]));
                at += issuers;
                if (at >= S) { at -= S; par ^= 1u; }
            }
            umma_commit_if<false>(lead, smem_u32(&done));     // (also after an expired wait)
        }
        odd ^= (uint32_t)((st + k_steps) / S) & 1u;
        st = (st + k_steps) % S;
    };
    if (warp == kProducer) {
        if (lane == 0) {
            for (int s = 0; s < S; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
            mbar_init(&done, issuers);
            mbar_init(&drained, kPlanners / 32);
            fence_mbar_init();
        }
        __syncwarp();
        for (int ks = 0; ks < early; ks++) {
            expect_more_if(lead, full0 + (uint32_t)(ks * 8), (uint32_t)shape.x_bytes);
            load_x(ks, ks);
        }
    }
    if (warp == kProducer + 1) {
        // TMEM first: a projection's block that came to this SM before would hold all of it
        // while it waits for this grid
        tmem_alloc(&tmem_slot, shape.cols);
        tmem_relinquish();
        grid_launch_dependents();
    }
    if (warp >= kProducer) {                  // the planners need neither barriers nor TMEM yet
        tc_fence_before();
        asm volatile("barrier.sync 2, %0;" ::"n"(kThreads - kPlanners) : "memory");
        tc_fence_after();
        if (direct) {
            if (warp == kProducer) fill(1, (int)blockIdx.y, 0);
            else multiply(1, 0);
        }
    }

    int n_here = 0, count = 0;
    long long first_block = 0;
    if (warp < kProducer) {
        if (tid == 0) present_mask = 0;
        auto end_of = [&](int u) { return a.off[u] + max(a.T[u], 0); };

        // utterances that end before the tile: ends ascend, kPlanners of them looked at at a time
        int lo = 0, hi = a.n_utt;
        while (hi - lo > kPlanners) {
            const int step = (hi - lo + kPlanners - 1) / kPlanners;
            const int u = lo + tid * step;
            const int n = plan_count(u < hi && end_of(u) <= tile0);
            if (n == 0) { hi = lo; break; }
            hi = min(hi, lo + n * step);          // the n-th looked at does not end before
            lo += (n - 1) * step + 1;
        }
        // the rest of them, and the utterances in the tile
        int n_seg = 0, ended = lo;
        for (int u0 = lo; u0 < a.n_utt; u0 += kPlanners) {
            const int u = u0 + tid;
            long long start = 0, end = 0;
            bool in = false, past = false, before = false;
            int ad = -1;
            if (u < a.n_utt) {
                start = a.off[u];
                past = start >= tile0 + n_rows;
                const int len = a.T[u], v = a.adapter[u];
                before = start + max(len, 0) <= tile0;
                in = !past && !before && len > 0;
                end = min(start + len - tile0, (long long)n_rows);
                ad = v >= 0 && v < a.n_adapters ? v : -1;
            }
            const uint32_t m = __ballot_sync(0xffffffffu, in);
            if (lane == 0) counts[warp] = __popc(m);
            plan_sync();
            int at = n_seg;
            for (int w = 0; w < kPlanners / 32; w++) {
                if (w < warp) at += counts[w];
                n_seg += counts[w];
            }
            at += __popc(m & ((1u << lane) - 1u));
            if (in && at < kMaxTile) {
                seg_start[at] = (uint16_t)max(start - tile0, 0LL);
                seg_end[at] = (uint16_t)end;
                seg_adapter[at] = ad;
            }
            ended += plan_count(before);
            if (u0 + kPlanners < a.n_utt && plan_count(past)) break;
        }
        n_seg = min(n_seg, kMaxTile);
        first_block = tile + (ended < tile0 ? ended : tile0);
        if (n_seg <= 32) {
            // by every warp for itself: each adapter once, and the row's
            const int v = lane < n_seg ? seg_adapter[lane] : -1;
            const int from = lane < n_seg ? seg_start[lane] : 0, to = lane < n_seg ? seg_end[lane] : 0;
            const uint32_t same = __match_any_sync(0xffffffffu, v);
            const bool first = v >= 0 && __ffs(same) - 1 == lane;
            const uint32_t firsts = __ballot_sync(0xffffffffu, first);
            const int at = __popc(firsts & ((1u << lane) - 1u));
            int slot = __shfl_sync(0xffffffffu, at, __ffs(same) - 1);
            // (utterances that overlap or are out of order must not lead out of the plan)
            count = (int)min((long long)__popc(firsts), max(p.blocks - first_block, 0LL));
            if (v < 0 || slot >= count) slot = -1;
            if (first && warp == 0) slots[at] = v;
            int mine = -1;
            for (int s = 0; s < n_seg; s++) {
                const int f = __shfl_sync(0xffffffffu, from, s), e = __shfl_sync(0xffffffffu, to, s);
                const int q = __shfl_sync(0xffffffffu, slot, s);
                if (local0 + tid >= f && local0 + tid < e) mine = q;
            }
            if (tid >= kRows) mine = -1;
            row_slot[tid] = mine;
            const uint32_t m = __reduce_or_sync(0xffffffffu, mine >= 0 ? 1u << mine : 0u);
            if (lane == 0 && m) atomicOr(&present_mask, m);
            plan_sync();
            const uint32_t pm = present_mask;
            n_here = __popc(pm);
            if (warp == 0 && lane < count) {
                const int before = __popc(pm & ((1u << lane) - 1u));
                here[pm >> lane & 1u ? before : count - 1 - (lane - before)] = (int16_t)lane;
            }
        } else {
            // each adapter once
            for (int i0 = 0; i0 < n_seg; i0 += kPlanners) {
                const int i = i0 + tid;
                int j = 0;                            // the first segment of this adapter
                if (i < n_seg) {
                    const int v = seg_adapter[i];
                    while (j + 4 <= i) {
                        const int4 q = *reinterpret_cast<const int4*>(seg_adapter + j);
                        if (q.x == v || q.y == v || q.z == v || q.w == v) break;
                        j += 4;
                    }
                    while (j < i && seg_adapter[j] != v) j++;
                }
                const bool first = i < n_seg && j == i && seg_adapter[i] >= 0;
                const uint32_t m = __ballot_sync(0xffffffffu, first);
                plan_sync();                      // counts are read
                if (lane == 0) counts[warp] = __popc(m);
                plan_sync();
                int at = count;
                for (int w = 0; w < kPlanners / 32; w++) {
                    if (w < warp) at += counts[w];
                    count += counts[w];
                }
                at += __popc(m & ((1u << lane) - 1u));
                if (first) slots[at] = seg_adapter[i];
                if (i < n_seg && j == i) seg_slot[i] = (int16_t)(first ? at : -1);
                plan_sync();
                if (i < n_seg && j != i) seg_slot[i] = seg_slot[j];
            }
            plan_sync();
            count = (int)min((long long)count, max(p.blocks - first_block, 0LL));
            {
                int l = 0, h = n_seg;                 // the last segment that starts at or before the row, if it has it
                while (l < h) {
                    const int m = (l + h) / 2;
                    if (seg_start[m] <= local0 + tid) l = m + 1; else h = m;
                }
                const int sl = tid < kRows && l > 0 && local0 + tid < seg_end[l - 1] ? seg_slot[l - 1] : -1;
                row_slot[tid] = sl < count ? sl : -1;
            }
            for (int i = tid; i < count; i += kPlanners) present[i] = 0;
            plan_sync();
            if (row_slot[tid] >= 0) present[row_slot[tid]] = 1;
            for (int i0 = 0; i0 < count; i0 += kPlanners) {
                plan_sync();
                const int i = i0 + tid;
                const bool is = i < count && present[i];
                const uint32_t m = __ballot_sync(0xffffffffu, is);
                if (lane == 0) counts[warp] = __popc(m);
                plan_sync();
                int at = n_here;
                for (int w = 0; w < kPlanners / 32; w++) {
                    if (w < warp) at += counts[w];
                    n_here += counts[w];
                }
                at += __popc(m & ((1u << lane) - 1u));
                if (is) here[at] = (int16_t)i;
                else if (i < count) here[count - 1 - (i - at)] = (int16_t)i;     // i - at: those absent before it
            }
        }
        plan_sync();
        if (row0 == tile0 && blockIdx.y == 0) {
            if (tid == 0) { p.tiles[tile].first = (int)first_block; p.tiles[tile].count = count; }
            for (int i = tid; i < count; i += kPlanners) {
                if (i < kInline) p.tiles[tile].adapter[i] = slots[i];
                p.adapter[first_block + i] = slots[i];
            }
        }
        if (blockIdx.y == 0 && warp * 32 < kRows) // this chunk's rows of each adapter
            for (int s = 0; s < count; s++) {
                const uint32_t mine = __ballot_sync(0xffffffffu, row_slot[tid] == s);
                if (lane == 0) p.owners[(first_block + s) * kOwnerWords + local0 / 32 + warp] = mine;
            }
        if (blockIdx.y == 0 && !direct)           // the others' blocks are zero in these rows
            for (int k = n_here; k < count; k++) {
                __half* out = p.t + ((first_block + here[k]) * p.tile + local0) * t_columns(rank);
                const int n = min(kRows, n_rows - local0) * t_columns(rank) / 8;
                for (int c = tid; c < n; c += kPlanners) reinterpret_cast<uint4*>(out)[c] = make_uint4(0u, 0u, 0u, 0u);
            }
        if (tid == 0) n_here_shared = n_here;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    n_here = n_here_shared;

    // adapters of a pass: two, or one where there are blocks for each
    const int side = n_here > (int)gridDim.y ? 2 : 1, stride = side * (int)gridDim.y, base0 = side * (int)blockIdx.y;
    if (warp == kProducer) {
        for (int base = base0; base < n_here && ok && !direct; base += stride) {
            const int n = uniform(min(side, n_here - base));
            const int ad0 = uniform(slots[here[base]]), ad1 = uniform(n > 1 ? slots[here[base + 1]] : 0);
            fill(n, ad0, ad1);
        }
        // no bulk copy may still be writing shared memory when the block exits: rows that
        // no adapter came for, and what the MMAs have not waited for
        for (int s = used; s < early; s++) {
            if (lane == 0) mbar_arrive(&full[s]);
            mbar_wait(&full[s], 0, a.err);
        }
        for (int s = 0; s < S; s++)
            if (issued >> s & 1u) mbar_wait(&full[s], s < st ? odd : odd ^ 1u, a.err);
        __syncwarp();
    } else if (warp > kProducer) {
        int pass = 0;
        for (int base = base0; base < n_here && !direct; base += stride, pass++) multiply(min(side, n_here - base), pass);
    } else {
        const uint32_t tmem = (uint32_t)uniform((int)tmem_slot);
        // an adapter's share, masked, as fp16 and what the rounding left: a row per lane
        const int r = warp * 32 + lane;
        const bool real = local0 + r < n_rows;
        const int mine = row_slot[r];
        // 16 columns of adapter e's sums: those of all issuers (the last sum may have fewer), and what came before
        const uint32_t total = tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)(issuers * acc_cols);
        auto sum_up = [&](int e, int c, int sum, float (&v)[16]) {
            const uint32_t from = tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)(e * n16 + c);
            const int parts = min(issuers, k_steps - sum * sum_steps);
            tmem_ld16(from, v);
            for (int w = 1; w < parts; w++) {
                float x[16];
                tmem_ld16(from + (uint32_t)(w * acc_cols), x);
#pragma unroll
                for (int i = 0; i < 16; i++) v[i] += x[i];
            }
            if (sum > 0) {
                float x[16];
                tmem_ld16(total + (uint32_t)(e * n16 + c), x);
#pragma unroll
                for (int i = 0; i < 16; i++) v[i] += x[i];
            }
        };
        auto store = [&](int e, int s) {
            const float sc = a.scale ? a.scale[slots[s]] : 1.f;
            __half* out = p.t + ((first_block + s) * p.tile + local0 + r) * t_columns(rank);
            for (int c = 0; c < rank; c += 16) {
                float v[16];
                sum_up(e, c, sums - 1, v);
                uint32_t hi[8], low[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const bool has = mine == s && c + 2 * i < rank;      // (the columns behind the rank hold anything)
                    const float v0 = has ? v[2 * i] * sc : 0.f, v1 = has ? v[2 * i + 1] * sc : 0.f;
                    const __half2 h = __floats2half2_rn(v0, v1);
                    const float2 f = __half22float2(h);
                    hi[i] = *reinterpret_cast<const uint32_t*>(&h);
                    low[i] = pack_half2(isinf(f.x) ? 0.f : v0 - f.x, isinf(f.y) ? 0.f : v1 - f.y);
                }
                if (!real) continue;
                const int r0 = c / kGroup * kGroup;
                uint4* o = reinterpret_cast<uint4*>(out + 2 * r0 + (c - r0));
                uint4* o2 = reinterpret_cast<uint4*>(out + 2 * r0 + group_width(rank, r0) + (c - r0));
                o[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                o[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                o2[0] = make_uint4(low[0], low[1], low[2], low[3]);
                o2[1] = make_uint4(low[4], low[5], low[6], low[7]);
            }
        };
        if (direct) {
            int s = 0;                        // this block's adapter among the tile's
            while (s < count && slots[s] != (int)blockIdx.y) s++;
            mbar_wait(&done, 0, a.err);
            __syncwarp();
            tc_fence_after();
            if (s < count && warp * 32 < kRows) store(0, s);
        }
        int pass = 0;
        for (int base = base0; base < n_here && !direct; base += stride, pass++) {
            for (int sum = 0; sum < sums - 1; sum++) {
                mbar_wait(&done, (uint32_t)(pass * sums + sum) & 1u, a.err);
                __syncwarp();
                tc_fence_after();
                if (warp * 32 < kRows)
                    for (int e = 0; e < min(side, n_here - base); e++)
                        for (int c = 0; c < rank; c += 16) {
                            float v[16];
                            sum_up(e, c, sum, v);
                            tmem_st16(total + (uint32_t)(e * n16 + c), v);
                        }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&drained);
            }
            mbar_wait(&done, (uint32_t)(pass * sums + sums - 1) & 1u, a.err);
            __syncwarp();
            tc_fence_after();
            if (warp * 32 < kRows)
                for (int e = 0; e < min(side, n_here - base); e++) store(e, here[base + e]);
            tc_fence_before();                // the accumulators are read before the next pass's products
            __syncwarp();
            if (lane == 0) mbar_arrive(&drained);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kProducer + 1) {
        tc_fence_after();
        tmem_dealloc(tmem_slot, shape.cols);
    }
}

template <int ROWS>
static int launch_rows(const LoraArgs& a, const LoraPlan& p, const CUtensorMap* x, int x_rows, cudaStream_t st) {
    auto kern = lora_shrink_kernel<ROWS>;
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!attr_set[dev & 63]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 218 * 1024) != cudaSuccess)
            return W2V_ERR_LAUNCH;
        attr_set[dev & 63] = true;
    }
    CUtensorMap tx, ta;
    const uint64_t xd[2] = {(uint64_t)a.K, (uint64_t)a.M}, xs[1] = {(uint64_t)a.lda * 2};
    int rc = W2V_OK;
    if (x && (x_rows == ROWS || (x_rows < ROWS && a.M <= x_rows))) {
        tx = *x;                               // (a box may be lower than a block that has no more rows)
    } else {
        x_rows = ROWS;
        rc = map_f16(&tx, a.x, 2, xd, xs, ROWS);
    }
    if (rc) return rc;
    const uint64_t ad[3] = {(uint64_t)a.K, (uint64_t)p.rank, (uint64_t)a.n_adapters};
    const uint64_t as[2] = {(uint64_t)a.K * 2, (uint64_t)a.K * 2 * p.rank};
    rc = map_f16(&ta, a.a, 3, ad, as, p.rank);
    if (rc) return rc;
    // few row chunks: a block per adapter that can meet there, side by side on the SMs
    const long long chunks = (a.M + ROWS - 1) / ROWS;
    long long most = p.tile;
    if (a.n_utt < most) most = a.n_utt;
    if (a.n_adapters < most) most = a.n_adapters;
    long long ny = 296 / chunks;
    if (ny > most) ny = most;
    if (ny < 1) ny = 1;
    ShrinkShape shape = shrink_shape(ROWS, p.rank, a.K / kStep, a.sums != 0);
    shape.x_bytes = x_rows * kStep * 2;
    shape.direct = chunks * a.n_adapters <= kDirect && shape.sums == 1;   // (sums are added once the plan is there)
    if (shape.direct) ny = a.n_adapters;
    kern<<<dim3((unsigned)chunks, (unsigned)ny), kThreads, shape.smem, st>>>(tx, ta, a, p, shape);
    return cudaPeekAtLastError() == cudaSuccess ? W2V_OK : W2V_ERR_LAUNCH;
}

int lora_shrink(const LoraArgs& a, const LoraPlan& p, const CUtensorMap* x, int x_rows, cudaStream_t st) {
    return p.tile % 128 == 0 && a.M >= 128 * 148 ? launch_rows<128>(a, p, x, x_rows, st) : launch_rows<64>(a, p, x, x_rows, st);
}

}  // namespace sg
}  // namespace w2v
