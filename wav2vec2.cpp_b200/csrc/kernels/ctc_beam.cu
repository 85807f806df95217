// CTC prefix beam search on the device: n best hypotheses of every utterance
// of a batch, resumable between calls.
//
// A beam is a prefix with the probabilities pb, pn of the paths that spell it
// and end in blank / in its last token.  With p the softmax row of a frame,
// total = pb + pn, and beam j the parent of beam i (i's prefix without its
// last token) when that is a beam too, a frame does
//   stay i:        pb' = total_i p[blank]
//                  pn' = (pn_i + (last_j == last_i ? pb_j : total_j)) p[last_i]
//   extend i by c: pn' = (c == last_i ? pb_i : total_i) p[c], unless that
//                  prefix is a beam (its stay has the contribution)
// and keeps the `width` candidates of largest pb' + pn'.
//
// Arithmetic.  Probabilities are held as 64-bit numbers relative to the best
// beam: each frame multiplies by exp(logit - row maximum) and rescales by a
// power of two (exact), so that no logarithm or exponential stands in the
// frame-to-frame chain.  The row maxima cancel; the powers of two are added up
// apart and the rows' sums multiplied (and rescaled alike), for the final score.
// Candidates below 2^-1000 of the frame's best are dropped, which also keeps
// every held value a normal number.  Selecting on 64-bit values matters:
// scores near the cut differ by less than 32 bits resolve after a few hundred
// frames.
//
// Candidates.  Tokens are ranked by p once per frame and beams are sorted by
// total.  The extension of beam i by the token of rank j is beaten by the
// (i + 1)(j + 1) - 1 pairs with no larger i and j, of which at most one per
// beam is not worth that much (the repeated token, which pb alone carries); a
// pair that is a beam already is outdone by that beam's stay.  So only pairs
// with (i + 1) j <= width can be kept: about width ln(width) candidates
// instead of width x V.
//
// Prefixes are nodes of a trie in the caller's state buffer, found again when
// a prefix that had been dropped is reached anew (its longer prefixes may have
// lived on): each beam carries a 64-bit filter of the tokens its node was ever
// extended by, and only on a hit the node's list of children is walked.
//
// Bound: the chain of frames, each a row of dependent instructions, shuffles and
// shared-memory round trips of few warps; a block holds an utterance, so 148 utterances
// take as long as one.  32 tokens, width 16: 1.05 us a frame (499 frames 0.51 ms, 64
// utterances of up to 499 0.53 ms); 94 tokens, width 100, 30 s: 2.0 us a frame, the
// extra on the barriers of eight search warps.  Hypotheses are found by reading the nodes of all
// frames so far: after 1500 frames of width 8 they add 27 us to a call, after 9000 146.
#include <float.h>

#include <algorithm>

#include "common.cuh"
#include "w2v_kernels.h"

namespace w2v {
namespace cb {

constexpr int kMaxWidth = 128;
constexpr int kMaxVocab = 1024;

typedef unsigned long long u64;

// One trie node; `head` is valid once its beam has been dropped (a live beam carries it).
struct Node {
    int parent, tok, head, next;
};

// Per-utterance state: this header, the beams' arrays, the nodes, the nodes' child filters.
struct Header {
    int frames, nb;
    u64 tag;             // of a started state, with the sizes it was laid out for
    long long exp2;      // power of two taken out of the beams so far
    long long z_exp2;    // and out of z
    double z;            // product of the rows' sums
};

// One beam, as the state keeps it between calls.
struct SavedBeam {
    double pb, pn;
    u64 mask;
    int node, last, len, pnode, par, head;
};

struct Layout {
    long long beams, nodes, masks, bytes;
};
__host__ __device__ inline Layout layout(int width, long long max_frames) {
    Layout l;
    const long long n = (long long)width * max_frames + 1;
    l.beams = sizeof(Header);
    l.nodes = (l.beams + (long long)width * (long long)sizeof(SavedBeam) + 15) / 16 * 16;
    l.masks = l.nodes + n * (long long)sizeof(Node);
    l.bytes = (l.masks + n * 8 + 255) / 256 * 256;
    return l;
}
__host__ __device__ inline u64 tag_of(int V, int blank, int width, int max_frames) {
    return 0x6265616d00000000ull ^ (u64)V << 52 ^ (u64)blank << 40 ^ (u64)width << 32 ^ (u64)max_frames;
}

struct Params {
    const float* logits;
    const long long* off;
    const int* T;
    int V, blank, width, max_frames, n_best, resume;
    uint8_t* state;
    int* ids;
    long long cap;
    int* n_ids;
    double* scores;
    int* err;
    int n_pairs;         // extension candidates (i, j): (i + 1) j <= width
    int slots;           // rows in the ring
    int copied;          // nodes that fit there for the hypotheses
};

// Tokens of rank 0 .. n_tok - 1 can extend a beam.
__host__ __device__ inline int n_tokens(int V, int width) { return V - 1 < width + 1 ? V - 1 : width + 1; }
__host__ __device__ inline int pairs_of(int i, int V, int width) {
    const int n = width / (i + 1) + 1;
    return n < V - 1 ? n : V - 1;
}

// A frame's row as the search needs it: by_rank[n_tok], key[V], id[V], p[V], z.
struct Ranked {
    double p;            // exp(logit - max), largest first (equal ones by token)
    int tok, pad;
};
struct Row {
    Ranked* by_rank;
    uint32_t* key;       // leading bits of p, 0 for blank and what cannot be emitted
    uint16_t* id;        // tokens of the keys, where not all are ranked
    double* p;           // by token
    double* z;           // the sum of p (0: nothing can be emitted)
};
__host__ __device__ inline int row_bytes(int V, int width) {
    return (n_tokens(V, width) * 16 + (V + 7) / 8 * 48 + (V + 1) * 8 + 15) / 16 * 16;
}
W2V_DEV Row row_at(uint8_t* base, int V, int n_tok) {
    Row r;
    r.by_rank = reinterpret_cast<Ranked*>(base);
    r.key = reinterpret_cast<uint32_t*>(base + n_tok * 16);
    r.id = reinterpret_cast<uint16_t*>(base + n_tok * 16 + (V + 7) / 8 * 32);
    r.p = reinterpret_cast<double*>(base + n_tok * 16 + (V + 7) / 8 * 48);
    r.z = r.p + V;
    return r;
}

// A candidate: its beam and, for an extension, its token + 1 (0: the stay).
W2V_DEV uint32_t pack_cand(int beam, int tok) { return (uint32_t)beam | (uint32_t)(tok + 1) << 8; }
W2V_DEV int beam_of(uint32_t c) { return (int)(c & 255u); }
W2V_DEV int token_of(uint32_t c) { return (int)(c >> 8) - 1; }

// The beams of a frame, one 16-byte word of each beam per array.
template <int MW>
struct Beams {
    struct Prob { double pb, total; } prob[MW];
    struct Info { int node, last, len, pnode; } info[MW];
    struct Link { uint32_t mask[2]; int head, par; } link[MW];   // mask: tokens (mod 64) the node was ever extended by
    double pn[MW];
};
// Candidates of a frame at most: MW stays and the sum of MW / i + 1 for i = 1 .. MW pairs, rounded up.
__host__ __device__ constexpr int max_live(int MW) {
    int n = MW;
    for (int i = 1; i <= MW; i++) n += MW / i + 1;
    return (n + 31) / 32 * 32;
}

template <int MW>
struct alignas(16) Shared {          // (what lies behind it is read 16 bytes at a time)
    uint32_t key32[max_live(MW)];    // leading bits of the values of the candidates in the running
    u64 key[max_live(MW)];           // the values
    Beams<MW> beams[2];
    struct Stay { double b, n; } stay[MW];       // the stays' pb', pn'
    struct Sel { u64 key; uint32_t cand, pad; } sel[MW];   // the new beams in order
    uint32_t cand[max_live(MW)];     // which candidates they are
    int slot[MW];                    // new place of an old beam that stays, -1: dropped
    int back[MW];                    // new beams whose node was found again
    int pair_at[MW];
    int n_live, n_back, expired;
    int place_sum;                   // of the candidates: less than all different ones add up to where values are equal
    uint32_t least_hi[8];
    // of the last frame, for the hypotheses
    int nb, cur;
    int n_nodes;
    long long exp2, z_exp2;
    double z;
};

// A logit as the search sees it: NaN cannot be emitted, +inf is the largest number.
W2V_DEV float clean(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }
W2V_DEV u64 bits_of(double x) { return (u64)__double_as_longlong(x); }   // positive numbers order as their bits
W2V_DEV double value_of(u64 k) { return __longlong_as_double((long long)k); }

// The best candidate of a frame is at least half and less than four times the
// best beam, which is held between 1 and 2: what is to be kept lies between
// 2^-1001 and 8.  Counted from 2^-1003, the exponent of such a value takes 10 bits,
// which leaves 22 of the fraction for a 32-bit key.
constexpr u64 kLeast = (u64)20 << 52;
W2V_DEV uint32_t leading(u64 k) { return (uint32_t)((k - kLeast) >> 30); }

// Row producer: one warp turns the logits of a frame into a Row.  Tokens are
// ranked by how many have larger leading bits, four keys a load; where two have
// the same, once more with the whole values and the id.  Of a large
// vocabulary only those are looked at that can be among the first n_tok: with m
// of a lane's tokens at or above the least m-th largest of all lanes, 32 m are.
template <bool LARGE>     // vocabularies of more than 64
W2V_DEV void make_row(const float* x, int V, int blank, int n_tok, float mx, const Row& r) {
    const int lane = threadIdx.x & 31, V4 = (V + 3) / 4;
    double z = 0.0;
    for (int v = lane; v < 4 * V4; v += 32) {
        const float l = v < V ? clean(x[v]) : -INFINITY;
        const double e = l == -INFINITY ? 0.0 : exp((double)l - (double)mx);
        if (v < V) r.p[v] = e;
        r.key[v] = v != blank && bits_of(e) >= kLeast ? leading(bits_of(e)) : 0;
        z += e;
    }
    for (int v = lane; v < n_tok; v += 32) r.by_rank[v] = Ranked{0.0, blank ? 0 : 1, 0};    // (fewer can be emitted)
    for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    __syncwarp();
    int n = V, n4 = V4;                  // keys to be ranked: all, or a list of them
    const bool some_only = LARGE && V > 192 && n_tok <= 128 && 2 * n_tok <= V;    // (no gain at 160, half the time at 400)
    if (some_only) {
        uint32_t top[4] = {0, 0, 0, 0};
        for (int v = lane; v < V; v += 32) {
            uint32_t k = r.key[v];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t hi = max(top[i], k);
                k = min(top[i], k);
                top[i] = hi;
            }
        }
        const int m = (n_tok + 31) / 32;
        const uint32_t least = max(__reduce_min_sync(0xffffffffu, top[m - 1]), 1u);
        n = 0;
        for (int v0 = 0; v0 < V; v0 += 32) {     // (the list stays behind what is still to be read)
            const int v = v0 + lane;
            const uint32_t k = v < V ? r.key[v] : 0;
            const uint32_t in = __ballot_sync(0xffffffffu, k >= least);
            const int at = n + __popc(in & ((1u << lane) - 1u));
            __syncwarp();
            if (k >= least) {
                r.key[at] = k;
                r.id[at] = (uint16_t)v;
            }
            n += __popc(in);
        }
        n4 = (n + 3) / 4;
        __syncwarp();
        if (lane < 4 * n4 - n) r.key[n + lane] = 0;
        __syncwarp();
    }
    int ranks = 0, some = 0;
    for (int a = lane; a < n; a += 32) {
        const uint32_t k = r.key[a];
        const int v = some_only ? r.id[a] : a;
        int c0 = 0, c1 = 0;
#pragma unroll 8
        for (int w = 0; w < n4; w++) {
            const uint4 q = reinterpret_cast<const uint4*>(r.key)[w];
            c0 += (q.x > k) + (q.y > k);
            c1 += (q.z > k) + (q.w > k);
        }
        if (k) {
            ranks += c0 + c1;
            some++;
            if (c0 + c1 < n_tok) r.by_rank[c0 + c1] = Ranked{r.p[v], v, 0};
        }
    }
    ranks = __reduce_add_sync(0xffffffffu, ranks);
    some = __reduce_add_sync(0xffffffffu, some);
    if (ranks != some * (some - 1) / 2) {
        // Among the same keys by the whole values and the id (the list's order).  Logits that came
        // from 16 bits, or that share a masked token's value, are here in nearly every frame.  Of
        // few tokens all values are compared, without a branch (32, 24 of them masked: 1.6 us a frame,
        // by the keys 1.9); of many by the keys, until n_tok are found to be better (400 tokens from
        // 16 bits, width 8: 4.5 us a frame, 1024: 7.3; by the values of all tokens 36 and 219).
        __syncwarp();
        if (!LARGE)
            for (int v = lane; v < V; v += 32) {
                const u64 e = bits_of(r.p[v]);
                int rank = 0;
                for (int w = 0; w < V; w++) {
                    const u64 f = bits_of(r.p[w]);
                    rank += w != blank && (w < v ? f >= e : f > e);
                }
                if (v != blank && rank < n_tok) r.by_rank[rank] = Ranked{value_of(e), v, 0};
            }
        else for (int a = lane; a < n; a += 32) {
            const uint32_t k = r.key[a];
            if (!k) continue;
            const int v = some_only ? r.id[a] : a;
            const double e = r.p[v];
            int rank = 0;
            for (int w = 0; w < n4 && rank < n_tok; w++) {
                const uint4 q = reinterpret_cast<const uint4*>(r.key)[w];
                rank += (q.x > k) + (q.y > k) + (q.z > k) + (q.w > k);
                const uint32_t same[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (same[i] == k) {
                        const int b = 4 * w + i;
                        const double f = r.p[some_only ? r.id[b] : b];
                        rank += b < a ? f >= e : f > e;
                    }
            }
            if (rank < n_tok) r.by_rank[rank] = Ranked{e, v, 0};
        }
    }
    if (lane == 0) *r.z = z;
    __syncwarp();
}

// 2^-1000 of the best.
W2V_DEV u64 pruned(u64 best) { return best > ((u64)1000 << 52) ? best - ((u64)1000 << 52) : 0; }
constexpr int kExtends = 1 << 16;    // in n_live, above the number: extensions among them (whatever multiple)

// Barrier of the NC search warps.
template <int NC>
W2V_DEV void search_sync() {
    if (NC == 1) __syncwarp();
    else asm volatile("barrier.sync 1, %0;" ::"n"(NC * 32) : "memory");
}
// Whether x holds for any thread of the search warps (a barrier too).
template <int NC>
W2V_DEV bool search_any(bool x) {
    int r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.s32 p, %1, 0;\n barrier.red.or.pred q, 1, %2, p;\n selp.s32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"((int)x), "n"(NC * 32)
        : "memory");
    return r != 0;
}

// How many of the keys are larger than k: 32 of every `step`, as long as they
// begin before n (keys behind the last are 0).
W2V_DEV int count_above(const uint32_t* keys, int n, int step, uint32_t k) {
    int c0 = 0, c1 = 0;
    for (int d = 0; d < n; d += step) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = reinterpret_cast<const uint4*>(keys + d)[i];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            c0 += (v[i].x > k) + (v[i].y > k);
            c1 += (v[i].z > k) + (v[i].w > k);
        }
    }
    return c0 + c1;
}

// NC search warps (the chain from frame to frame; beam i is thread i's) and
// NP row producers (frame t: warp t % NP), a ring of rows between them; one more
// warp multiplies the rows' sums, which nothing in the chain needs.
template <int NC, int NP, int MW>
__global__ void __launch_bounds__((NC + NP + 1) * 32, 1) ctc_beam_kernel(Params p) {
    constexpr int NT = NC * 32;
    constexpr int kPairs = (max_live(MW) - MW + NT - 1) / NT;       // of a thread
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ uint64_t full[2 * NP], empty[2 * NP];
    Shared<MW>& s = *reinterpret_cast<Shared<MW>*>(smem_raw);
    uint32_t* bits = reinterpret_cast<uint32_t*>(smem_raw + sizeof(Shared<MW>));   // [width][words]
    const int u = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int W = p.width, V = p.V, n_tok = n_tokens(V, W), words = (V + 31) / 32;
    uint8_t* rows = smem_raw + sizeof(Shared<MW>) + (W * words * 4 + 15) / 16 * 16;
    const Layout lay = layout(W, p.max_frames);
    uint8_t* st = p.state + (long long)u * lay.bytes;
    Header* hdr = reinterpret_cast<Header*>(st);
    SavedBeam* saved = reinterpret_cast<SavedBeam*>(st + lay.beams);
    Node* nodes = reinterpret_cast<Node*>(st + lay.nodes);
    u64* masks = reinterpret_cast<u64*>(st + lay.masks);

    const int T = p.T[u] > 0 ? p.T[u] : 0;
    int frames = 0, nb = 1;
    long long exp2 = 0;
    const u64 tag = tag_of(V, p.blank, W, p.max_frames);
    bool refused = p.resume && hdr->tag != tag;      // not a state of such a search
    if (p.resume && !refused) {
        frames = hdr->frames;
        nb = hdr->nb;
        exp2 = hdr->exp2;
    }
    refused = refused || T > p.max_frames - frames;
    if (refused && tid == 0) report_error(p.err, kErrBadArgs);
    if (tid < 2 * NP) {
        mbar_init(&full[tid], 1);
        mbar_init(&empty[tid], 2);       // search warps and the product of sums
        fence_mbar_init();
    }
    if (tid == 0) {
        s.n_live = 0;
        s.n_back = 0;
        s.expired = 0;
        s.place_sum = 0;
    }
    __syncthreads();                     // the row producers need no more

    const int n_frames = refused ? 0 : T;
    const float* x = p.logits + p.off[u] * V;
    const int rbytes = row_bytes(V, W);
    if (warp == NC + NP) {
        double z = 1.0;
        long long z_exp2 = 0;
        bool ok = true;
        if (p.resume && !refused) {
            z = hdr->z;
            z_exp2 = hdr->z_exp2;
        }
        int sl = 0;
        uint32_t odd = 0;
        for (int t = 0; t < n_frames && ok; t++) {
            ok = __all_sync(0xffffffffu, mbar_wait(&full[sl], odd, p.err));
            if (!ok) break;
            const double row_z = *row_at(rows + sl * rbytes, V, n_tok).z;
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[sl]);
            if (row_z > 0.0) {               // (0: no hypothesis is left)
                const u64 v = bits_of(z * row_z);
                const int e = (int)(v >> 52) - 1023;
                z = value_of(v - ((u64)e << 52));
                z_exp2 += e;
            }
            if (++sl == p.slots) { sl = 0; odd ^= 1u; }
        }
        if (lane == 0) {
            s.z = z;
            s.z_exp2 = z_exp2;
            if (!refused && ok) {
                hdr->z = z;
                hdr->z_exp2 = z_exp2;
            }
        }
    } else if (warp >= NC) {
        int sl = warp - NC;              // slot of the frame, and whether the ring's rounds so far are odd
        uint32_t odd = 0;
        for (int t = warp - NC; t < n_frames; t += NP) {
            const float* row = x + (long long)t * V;
            float mx = -INFINITY;
            for (int v = lane; v < V; v += 32) mx = fmaxf(mx, clean(row[v]));
            for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[sl], odd ^ 1u, p.err))) break;
            make_row<(NP > 2)>(row, V, p.blank, n_tok, mx, row_at(rows + sl * rbytes, V, n_tok));
            if (lane == 0) mbar_arrive(&full[sl]);
            sl += NP;
            if (sl >= p.slots) { sl -= p.slots; odd ^= 1u; }
        }
    } else {
        for (int i = tid; i < W * words; i += NT) bits[i] = 0;
        for (int i = tid; i < max_live(MW); i += NT) s.key32[i] = 0;
        if (warp == 0) {                 // where each beam's pairs start
            int before = 0;
            for (int i0 = 0; i0 < MW; i0 += 32) {
                const int n = i0 + lane < W ? pairs_of(i0 + lane, V, W) : 0;
                int incl = n;
                for (int d = 1; d < 32; d <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, incl, d);
                    if (lane >= d) incl += v;
                }
                s.pair_at[i0 + lane] = before + incl - n;
                before += __shfl_sync(0xffffffffu, incl, 31);
            }
        }
        double my_pb = 0.0, my_pn = 0.0, my_total = 0.0;     // this thread's beam
        int my_last = -1, my_par = -1;
        search_sync<NC>();
        if (tid < nb && !refused) {
            SavedBeam v{1.0, 0.0, 0, 0, -1, 0, -1, -1, -1};
            if (p.resume) v = saved[tid];
            else nodes[0] = Node{-1, -1, -1, -1};
            my_pb = v.pb;
            my_pn = v.pn;
            my_total = my_pb + my_pn;
            my_last = v.last;
            my_par = v.par;
            s.beams[0].prob[tid] = {my_pb, my_total};
            s.beams[0].pn[tid] = my_pn;
            s.beams[0].info[tid] = {v.node, v.last, v.len, v.pnode};
            s.beams[0].link[tid] = {{(uint32_t)v.mask, (uint32_t)(v.mask >> 32)}, v.head, v.par};
            if (my_par >= 0) atomicOr(&bits[my_par * words + (my_last >> 5)], 1u << (my_last & 31));
        }
        int pi[kPairs], pj[kPairs];      // this thread's extensions (beam, rank), beam MW: none
#pragma unroll
        for (int e = 0; e < kPairs; e++) {
            const int c = e * NT + tid;
            int i = 0;                   // the last beam whose pairs start at or before c
#pragma unroll
            for (int d = MW / 2; d; d /= 2)
                if (i + d < W && s.pair_at[i + d] <= c) i += d;
            pi[e] = c < p.n_pairs ? i : MW;
            pj[e] = c < p.n_pairs ? c - s.pair_at[i] : 0;
        }
        search_sync<NC>();
        int sl = 0, cur = 0;
        uint32_t odd = 0;
        bool ready = false;              // the frame's row was seen to be complete
        for (int t = 0; t < n_frames; t++) {
            if (!ready && !mbar_wait(&full[sl], odd, p.err)) s.expired = 1;
            const Row r = row_at(rows + sl * rbytes, V, n_tok);
            const Beams<MW>& b = s.beams[cur];
            Beams<MW>& n = s.beams[cur ^ 1];
            // all that the frame's candidates need, before anything is stored
            Ranked kr[kPairs];
            typename Beams<MW>::Prob kq[kPairs];
            int kl[kPairs];
            uint32_t kw[kPairs];
#pragma unroll
            for (int e = 0; e < kPairs; e++) {
                const int i = pi[e] < W ? pi[e] : 0;     // beams from nb on hold something, and are left out below
                kr[e] = r.by_rank[pj[e]];
                kq[e] = b.prob[i];
                kl[e] = b.info[i].last;
                kw[e] = bits[i * words + (kr[e].tok >> 5)] >> (kr[e].tok & 31);
            }
            const int me = tid < W ? tid : 0, up = my_par >= 0 ? my_par : 0;
            const Ranked k0 = r.by_rank[0], k1 = r.by_rank[n_tok > 1 ? 1 : 0];
            const double p_blank = r.p[p.blank], p_last = r.p[my_last >= 0 ? my_last : 0];
            const auto above = b.prob[up];
            const int above_last = b.info[up].last;
            const uint32_t w0 = bits[me * words + (k0.tok >> 5)] >> (k0.tok & 31);
            const uint32_t w1 = bits[me * words + (k1.tok >> 5)] >> (k1.tok & 31);
            // the stays, and each beam's best candidate: `width` different ones, so the
            // least of them bounds from below what can be kept
            u64 stay = 0, most = ~(u64)0;
            double stay_b = 0.0, stay_n = 0.0;
            if (tid < nb) {
                const double from = my_par >= 0 ? my_pn + (above_last == my_last ? above.pb : above.total) : my_pn;
                stay_b = my_total * p_blank;
                stay_n = my_last >= 0 ? from * p_last : 0.0;
                stay = bits_of(stay_b + stay_n);
                most = stay;
                // no more than two looked at: the likeliest token is as a rule neither a beam's already nor the beam's last
                const u64 e0 = bits_of((k0.tok == my_last ? my_pb : my_total) * k0.p);
                const u64 e1 = bits_of((k1.tok == my_last ? my_pb : my_total) * k1.p);
                if (!(w0 & 1u) && e0 > most) most = e0;
                if (!(w1 & 1u) && e1 > most) most = e1;
                s.stay[tid] = {stay_b, stay_n};
                s.slot[tid] = -1;
            }
            uint32_t least = __reduce_min_sync(0xffffffffu, (uint32_t)(most >> 32));
            if (NC > 1 && lane == 0) s.least_hi[warp] = least;
            // the extensions
            u64 key[kPairs];
            uint32_t cand[kPairs];
#pragma unroll
            for (int e = 0; e < kPairs; e++) {
                cand[e] = pack_cand(pi[e], kr[e].tok);
                const u64 v = bits_of((kr[e].tok == kl[e] ? kq[e].pb : kq[e].total) * kr[e].p);
                key[e] = pi[e] < nb && !(kw[e] & 1u) ? v : 0;
            }
            search_sync<NC>();
            if (s.expired) break;
            if (NC > 1) {
#pragma unroll
                for (int i = 0; i < NC; i++) least = min(least, s.least_hi[i]);
            }
            if (nb < W) least = 0;
            // those in the running
            uint32_t in[kPairs + 1];
            int total_in = 0;
#pragma unroll
            for (int e = 0; e <= kPairs; e++) {
                const u64 k = e < kPairs ? key[e < kPairs ? e : 0] : stay;
                in[e] = __ballot_sync(0xffffffffu, k >= kLeast && (uint32_t)(k >> 32) >= least);
                total_in += __popc(in[e]);
            }
            // Only stays, in the order they had (most blank frames): the beams keep their places,
            // tokens and nodes, and no more than their probabilities change.
            uint32_t extends = 0;
#pragma unroll
            for (int e = 0; e < kPairs; e++) extends |= in[e];
            auto unchanged = [&](u64 best, u64 next) {
                return tid >= nb || (stay >= kLeast && stay >= pruned(best) && (tid + 1 == nb || stay >= next));
            };
            auto keep_places = [&](u64 best) {
                const int e2 = (int)(best >> 52) - 1023;
                const double scale = value_of((u64)(1023 - e2) << 52);
                if (tid < nb) {
                    my_pb = stay_b * scale;
                    my_pn = stay_n * scale;
                    my_total = my_pb + my_pn;
                    s.beams[cur].prob[tid] = {my_pb, my_total};
                    s.beams[cur].pn[tid] = my_pn;
                }
                if (tid == 0) mbar_arrive(&empty[sl]);
                exp2 += e2;
                if (++sl == p.slots) { sl = 0; odd ^= 1u; }
                ready = t + 1 < n_frames && mbar_try_wait(&full[sl], odd);
            };
            if (NC == 1 && nb && !extends) {
                const u64 best = __shfl_sync(0xffffffffu, stay, 0), next = __shfl_down_sync(0xffffffffu, stay, 1);
                if (__all_sync(0xffffffffu, unchanged(best, next))) {
                    keep_places(best);
                    __syncwarp();
                    continue;
                }
            }
            if (NC == 1 || total_in) {
                int at = 0;
                if (NC > 1) {
                    if (lane == 0) at = atomicAdd(&s.n_live, total_in | (extends ? kExtends : 0)) & (kExtends - 1);
                    at = __shfl_sync(0xffffffffu, at, 0);
                }
#pragma unroll
                for (int e = 0; e <= kPairs; e++) {
                    if (in[e] >> lane & 1u) {
                        const int pos = at + __popc(in[e] & ((1u << lane) - 1u));
                        const u64 k = e < kPairs ? key[e < kPairs ? e : 0] : stay;
                        s.key[pos] = k;
                        s.key32[pos] = leading(k);
                        s.cand[pos] = e < kPairs ? cand[e < kPairs ? e : 0] : pack_cand(tid, -1);
                    }
                    at += __popc(in[e]);
                }
            }
            search_sync<NC>();
            const int live = NC == 1 ? total_in : s.n_live & (kExtends - 1);
            if (NC > 1 && nb && live == s.n_live) {
                const u64 best = bits_of(s.stay[0].b + s.stay[0].n);
                const u64 next = tid + 1 < nb ? bits_of(s.stay[tid + 1].b + s.stay[tid + 1].n) : 0;
                if (!search_any<NC>(!unchanged(best, next))) {
                    for (int a = tid; a < live; a += NT) s.key32[a] = 0;
                    if (tid == 0) s.n_live = 0;
                    keep_places(best);
                    search_sync<NC>();
                    continue;
                }
            }
            // their places in order: how many have larger leading bits (which decide but for one
            // frame in some hundreds)
            auto put = [&](int c, int a) {
                if (c >= W) return;
                const uint32_t cd = s.cand[a];
                s.sel[c] = {s.key[a], cd, 0};
                if (token_of(cd) < 0) s.slot[beam_of(cd)] = c;
            };
            int places = 0;
            if (NC > 1 && 2 * live <= NT) {      // two threads per candidate, 32 of the others in turn
                const int a = tid >> 1;
                int c = 0;
                if (warp * 16 < live) {
                    c = count_above(s.key32 + (tid & 1) * 32, live - (tid & 1) * 32, 64, s.key32[a]);
                    c += __shfl_xor_sync(0xffffffffu, c, 1);
                }
                if (a < live && !(tid & 1)) {
                    places = c;
                    put(c, a);
                }
            } else {
                for (int a = tid; a < live; a += NT) {
                    const int c = count_above(s.key32, live, 32, s.key32[a]);
                    places += c;
                    put(c, a);
                }
            }
            // equal ones take one place: the places add up to less than 0 + 1 + .. + live - 1
            auto all_differ = [&]() {
                places = __reduce_add_sync(0xffffffffu, places);
                if (NC > 1 && lane == 0) atomicAdd(&s.place_sum, places);
                search_sync<NC>();
                return (NC > 1 ? s.place_sum : places) == live * (live - 1) / 2;
            };
            if (!all_differ()) {
                // by the whole values
                search_sync<NC>();
                if (tid < nb) s.slot[tid] = -1;
                if (tid == 0) s.place_sum = 0;
                search_sync<NC>();
                places = 0;
                for (int a = tid; a < live; a += NT) {
                    const u64 k = s.key[a];
                    int c = 0;
#pragma unroll 8
                    for (int d = 0; d < live; d++) c += s.key[d] > k;
                    places += c;
                    put(c, a);
                }
                if (!all_differ()) {
                    // and the rule for equal ones: stays first, then by beam and token
                    if (tid < nb) s.slot[tid] = -1;
                    search_sync<NC>();
                    auto order = [&](uint32_t c) {
                        return token_of(c) < 0 ? beam_of(c) : W + beam_of(c) * V + token_of(c);
                    };
                    for (int a = tid; a < live; a += NT) {
                        const u64 k = s.key[a];
                        const int o = order(s.cand[a]);
                        int c = 0;
                        for (int d = 0; d < live; d++) c += s.key[d] > k || (s.key[d] == k && order(s.cand[d]) < o);
                        put(c, a);
                    }
                    search_sync<NC>();
                }
            }
            // the new beams, but those below 2^-1000 of the best
            int nn = min(live, W);
            const u64 best = nn ? s.sel[0].key : 0;
            const int e2 = nn ? (int)(best >> 52) - 1023 : 0;
            const double scale = value_of((u64)(1023 - e2) << 52);
            const u64 floor = pruned(best);
            while (nn && s.sel[nn - 1].key < floor) nn--;
            const int my_slot = tid < nb ? s.slot[tid] : 0;
            const bool drops = tid < nb && (uint32_t)my_slot >= (uint32_t)nn;
            if (tid < nb && my_par >= 0) bits[my_par * words + (my_last >> 5)] = 0;
            int fresh = -1;          // the old beam whose new child this thread's beam is
            int my_node = 0, my_pnode = 0;
            if (tid < nn) {
                const auto c = s.sel[tid];
                const int i = beam_of(c.cand), tk = token_of(c.cand);
                const bool stays = tk < 0;
                const auto info = b.info[i];
                const auto link = b.link[i];
                const auto held = s.stay[i];
                const int from = stays ? link.par : i;           // old place of the parent
                int par = s.slot[from >= 0 ? from : 0];
                if (from < 0 || par >= nn) par = -1;
                uint32_t mask0 = link.mask[0], mask1 = link.mask[1];
                int head = link.head;
                my_node = info.node;
                if (!stays) {
                    int id = -1;
                    if ((tk & 32 ? mask1 : mask0) >> (tk & 31) & 1u)
                        for (id = head; id >= 0 && nodes[id].tok != tk; id = nodes[id].next) {}
                    if (id >= 0) {   // reached again after it was dropped
                        head = nodes[id].head;
                        mask0 = (uint32_t)masks[id];
                        mask1 = (uint32_t)(masks[id] >> 32);
                        s.back[atomicAdd(&s.n_back, 1)] = tid;
                    } else {
                        id = 1 + (frames + t) * W + tid;
                        head = -1;
                        mask0 = mask1 = 0;
                        fresh = i;
                    }
                    my_node = id;
                }
                my_pnode = stays ? info.pnode : info.node;
                my_last = stays ? info.last : tk;
                my_pb = stays ? held.b * scale : 0.0;
                my_pn = (stays ? held.n : value_of(c.key)) * scale;
                my_total = my_pb + my_pn;
                my_par = par;
                n.prob[tid] = {my_pb, my_total};
                n.pn[tid] = my_pn;
                n.info[tid] = {my_node, my_last, info.len + !stays, my_pnode};
                n.link[tid] = {{mask0, mask1}, head, par};
            }
            for (int a = tid; a < live; a += NT) s.key32[a] = 0;
            search_sync<NC>();
            if (tid == 0) {
                mbar_arrive(&empty[sl]);
                s.n_live = 0;
                s.place_sum = 0;
            }
            const int nback = s.n_back;
            // children join their parents' lists (a parent that drops: its old place's), and mark them
            if (fresh >= 0) {
                auto& parent = my_par >= 0 ? n.link[my_par] : s.beams[cur].link[fresh];
                nodes[my_node] = Node{my_pnode, my_last, -1, atomicExch(&parent.head, my_node)};
                atomicOr(&parent.mask[my_last >> 5 & 1], 1u << (my_last & 31));
            }
            if (tid < nn) {
                if (nback && my_par < 0)
                    for (int i = 0; i < nback; i++)
                        if (n.info[s.back[i]].node == my_pnode) n.link[tid].par = my_par = s.back[i];
                if (my_par >= 0) atomicOr(&bits[my_par * words + (my_last >> 5)], 1u << (my_last & 31));
            }
            search_sync<NC>();
            if (drops) {
                const int id = b.info[tid].node;
                nodes[id].head = b.link[tid].head;
                masks[id] = (u64)b.link[tid].mask[1] << 32 | b.link[tid].mask[0];
            }
            if (tid == 0) s.n_back = 0;
            exp2 += e2;
            nb = nn;
            cur ^= 1;
            if (++sl == p.slots) { sl = 0; odd ^= 1u; }
            ready = t + 1 < n_frames && mbar_try_wait(&full[sl], odd);
        }
        search_sync<NC>();
        const bool failed = s.expired != 0;  // a wait ran out (reported by mbar_wait)
        if (tid == 0) {
            s.nb = refused || failed ? 0 : nb;
            s.cur = cur;
            s.exp2 = exp2;
            s.n_nodes = refused || failed ? 0 : 1 + (frames + T) * W;
            if (failed) hdr->tag = 0;
        }
        // state for the next call
        if (!refused && !failed) {
            if (tid == 0) {
                hdr->frames = frames + T;
                hdr->nb = nb;
                hdr->tag = tag;
                hdr->exp2 = exp2;
            }
            if (tid < nb) {
                const auto info = s.beams[cur].info[tid];
                const auto link = s.beams[cur].link[tid];
                saved[tid] = SavedBeam{my_pb, my_pn, (u64)link.mask[1] << 32 | link.mask[0], info.node, info.last, info.len, info.pnode, link.par, link.head};
            }
        }
    }
    if (p.n_best == 0) return;
    __syncthreads();
    // hypotheses, best first
    constexpr int kWarps = NC + NP + 1;
    const Beams<MW>& b = s.beams[s.cur];
    const int have = s.nb < p.n_best ? s.nb : p.n_best;
    for (int h = warp; h < p.n_best; h += kWarps) {
        const int len = h < have ? b.info[h].len : 0;
        int* out = p.ids + ((long long)u * p.n_best + h) * p.cap;
        for (long long i = len + lane; i < p.cap; i += 32) out[i] = -1;
    }
    // A lane each walks from its hypothesis' node up, through a copy of the nodes in shared memory, newest
    // first (a node's parent is older): a step from global memory takes some 300 ns, and a stream's call of few
    // frames would spend more on the walk than on the frames.
    static_assert(kWarps * 32 >= MW, "a lane for each hypothesis");
    const int h = lane * kWarps + warp;
    int id = -1, left = 0;               // left: tokens still to be found
    int* out = nullptr;
    if (h < p.n_best) {
        const long long at = (long long)u * p.n_best + h;
        const int len = h < have ? b.info[h].len : -1;
        p.n_ids[at] = len;
        p.scores[at] = h < have ? log(b.prob[h].total) - log(s.z) + (double)(s.exp2 - s.z_exp2) * 0.69314718055994530942
                                : -INFINITY;
        if (len > 0) {
            id = b.info[h].node;
            left = len;
            out = p.ids + at * p.cap;
        }
    }
    int2* copy = reinterpret_cast<int2*>(rows);
    for (int hi = s.n_nodes, lo; __syncthreads_or(left > 0) && hi > 0; hi = lo) {
        lo = max(hi - p.copied, 0);
        constexpr int kStep = kWarps * 32;
        const int n = hi - lo;               // (counted from lo: node numbers go up to the end of an int)
        for (int k0 = tid; k0 < n; k0 += 8 * kStep) {
            int2 v[8];
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (k0 + e * kStep < n) v[e] = *reinterpret_cast<const int2*>(nodes + lo + k0 + e * kStep);
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (k0 + e * kStep < n) copy[k0 + e * kStep] = v[e];
        }
        __syncthreads();
        while (left > 0 && id >= lo && id < hi) {
            const int2 v = copy[id - lo];            // parent, token
            if (--left < p.cap) out[left] = v.y;
            id = v.x;
        }
    }
}

template <int NC, int NP, int MW>
static int launch(Params p, int n_utt, cudaStream_t st) {
    const long long fixed = (long long)sizeof(Shared<MW>) + (p.width * ((p.V + 31) / 32) * 4 + 15) / 16 * 16;
    const long long row = row_bytes(p.V, p.width);
    p.slots = fixed + 2 * NP * row <= 200 * 1024 ? 2 * NP : NP;
    // room for the nodes too, no more than leaves as many blocks on an SM as there are
    long long smem = fixed + p.slots * row;
    const long long all = fixed + ((long long)p.width * p.max_frames + 1) * (long long)sizeof(int2);
    if (p.n_best) smem = std::max(smem, std::min(all, 200 * 1024LL / ((n_utt + 147) / 148)));
    p.copied = (int)((smem - fixed) / (long long)sizeof(int2));
    static bool attr[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    auto kern = ctc_beam_kernel<NC, NP, MW>;
    if (!attr[dev & 63]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024) != cudaSuccess)
            return W2V_ERR_LAUNCH;
        attr[dev & 63] = true;
    }
    kern<<<n_utt, (NC + NP + 1) * 32, smem, st>>>(p);
    return cudaPeekAtLastError() == cudaSuccess ? W2V_OK : W2V_ERR_LAUNCH;
}

}  // namespace cb
}  // namespace w2v

using namespace w2v::cb;

extern "C" long long w2v_ctc_beam_state_bytes(int n_utt, int V, int width, int max_frames) {
    if (n_utt < 0 || V < 2 || V > kMaxVocab || width < 1 || width > kMaxWidth || max_frames < 1 ||
        (long long)width * max_frames >= 0x7fffffffLL)
        return -1;
    const long long bytes = layout(width, max_frames).bytes;
    return n_utt <= 0x7fffffffffffffffLL / bytes ? n_utt * bytes : -1;
}

extern "C" int w2v_ctc_beam(const float* logits, const long long* off, const int* T, int n_utt, int V, int blank,
                            int width, int max_frames, int resume, void* state, long long state_bytes, int n_best,
                            int* ids, long long cap, int* n_ids, double* scores, int* err, void* stream) {
    const long long need = w2v_ctc_beam_state_bytes(n_utt, V, width, max_frames);
    if (need < 0 || blank < 0 || blank >= V || n_best < 0 || n_best > width) return W2V_ERR_ARGS;
    if (n_utt == 0) return W2V_OK;
    if (!logits || !off || !T || !state || (reinterpret_cast<uintptr_t>(state) & 15)) return W2V_ERR_ARGS;
    if (n_best && (!ids || !n_ids || !scores || cap < 1)) return W2V_ERR_ARGS;
    if (state_bytes < need) return W2V_ERR_CAPACITY;
    Params p;
    p.logits = logits;
    p.off = off;
    p.T = T;
    p.V = V;
    p.blank = blank;
    p.width = width;
    p.max_frames = max_frames;
    p.n_best = n_best;
    p.resume = resume != 0;
    p.state = reinterpret_cast<uint8_t*>(state);
    p.ids = ids;
    p.cap = cap;
    p.n_ids = n_ids;
    p.scores = scores;
    p.err = err;
    p.n_pairs = 0;
    for (int i = 0; i < width; i++) p.n_pairs += pairs_of(i, V, width);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    // Up to 32 beams one warp searches, without barriers, and takes about a microsecond a frame;
    // a row of 32 tokens costs a producer half of that, one of 200 ten times as much.  More beams take
    // eight warps, whatever their number (32 tokens, 8 utterances: width 32 1.4 us a frame, 33 1.8, 64
    // 1.9, 100 2.2, 128 2.4; one warp with several beams a lane has not been measured).
    if (width <= 32) return V <= 64 ? launch<1, 2, 32>(p, n_utt, st) : launch<1, 7, 32>(p, n_utt, st);
    return launch<8, 7, 128>(p, n_utt, st);
}
