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
// frame-to-frame chain.  The row maxima cancel, the powers of two and the
// logarithms of the rows' sums are added up apart and enter the final score.
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
#include <float.h>

#include "common.cuh"
#include "w2v_kernels.h"

namespace w2v {
namespace cb {

constexpr int kMaxWidth = 128;
constexpr int kMaxVocab = 1024;
constexpr int kThreads = 256;

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
    double log_z;        // sum of the logarithms of the rows' sums
};

struct Beams {           // structure of arrays, `width` long each
    double *pb, *pn;
    u64* mask;
    int *node, *last, *len, *pnode, *par, *head;
};
constexpr int kBeamBytes = 3 * 8 + 6 * 4;

struct Layout {
    long long beams, nodes, masks, bytes;
};
__host__ __device__ inline Layout layout(int width, long long max_frames) {
    Layout l;
    const long long n = (long long)width * max_frames + 1;
    l.beams = sizeof(Header);
    l.nodes = (l.beams + (long long)width * kBeamBytes + 15) / 16 * 16;
    l.masks = l.nodes + n * (long long)sizeof(Node);
    l.bytes = (l.masks + n * 8 + 255) / 256 * 256;
    return l;
}
__host__ __device__ inline Beams beams_at(void* base, int width) {
    Beams b;
    b.pb = reinterpret_cast<double*>(base);
    b.pn = b.pb + width;
    b.mask = reinterpret_cast<u64*>(b.pn + width);
    b.node = reinterpret_cast<int*>(b.mask + width);
    b.last = b.node + width;
    b.len = b.last + width;
    b.pnode = b.len + width;
    b.par = b.pnode + width;
    b.head = b.par + width;
    return b;
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
};

// Tokens of rank 0 .. n_tok - 1 can extend a beam.
__host__ __device__ inline int n_tokens(int V, int width) { return V - 1 < width + 1 ? V - 1 : width + 1; }
__host__ __device__ inline int pairs_of(int i, int V, int width) {
    const int n = width / (i + 1) + 1;
    return n < V - 1 ? n : V - 1;
}

struct Smem {
    double* p;           // [V] exp(logit - max)
    double* sp;          // [n_tok] the same by rank
    u64* key;            // [width + n_pairs]
    uint32_t* order;     // [width + n_pairs] order among equal values: stays, then (beam, token)
    uint32_t* bits;      // [width][words] tokens whose extension of the beam is a beam
    int* stok;           // [n_tok] token by rank
    int* sel;            // [width] candidate of each new beam
    int* slot;           // [width] new place of an old beam, -1: dropped
    int* back;           // [width] new beams whose node was found again
    uint16_t* pair;      // [n_pairs] beam in the high byte, rank in the low
    Beams b[2];
    int words;
};
__host__ __device__ inline long long smem_layout(Smem* s, uint8_t* base, int V, int width, int n_pairs) {
    const int nt = n_tokens(V, width), nc = width + n_pairs, words = (V + 31) / 32;
    long long o = 0;
    auto take = [&](long long bytes) { const long long at = o; o += (bytes + 15) / 16 * 16; return base + at; };
    uint8_t* p = take(8LL * V);
    uint8_t* sp = take(8LL * nt);
    uint8_t* key = take(8LL * nc);
    uint8_t* b0 = take((long long)width * kBeamBytes);
    uint8_t* b1 = take((long long)width * kBeamBytes);
    uint8_t* order = take(4LL * nc);
    uint8_t* bits = take(4LL * width * words);
    uint8_t* stok = take(4LL * nt);
    uint8_t* sel = take(4LL * width);
    uint8_t* slot = take(4LL * width);
    uint8_t* back = take(4LL * width);
    uint8_t* pair = take(2LL * n_pairs);
    if (s) {
        s->p = reinterpret_cast<double*>(p);
        s->sp = reinterpret_cast<double*>(sp);
        s->key = reinterpret_cast<u64*>(key);
        s->b[0] = beams_at(b0, width);
        s->b[1] = beams_at(b1, width);
        s->order = reinterpret_cast<uint32_t*>(order);
        s->bits = reinterpret_cast<uint32_t*>(bits);
        s->stok = reinterpret_cast<int*>(stok);
        s->sel = reinterpret_cast<int*>(sel);
        s->slot = reinterpret_cast<int*>(slot);
        s->back = reinterpret_cast<int*>(back);
        s->pair = reinterpret_cast<uint16_t*>(pair);
        s->words = words;
    }
    return o;
}

// A logit as the search sees it: NaN cannot be emitted, +inf is the largest number.
W2V_DEV float clean(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

__global__ void __launch_bounds__(kThreads) ctc_beam_kernel(Params p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ float red_f[kThreads / 32];
    __shared__ double red_d[kThreads / 32];
    __shared__ u64 best_key;
    __shared__ int n_new, n_back;
    Smem s;
    smem_layout(&s, smem_raw, p.V, p.width, p.n_pairs);
    const int u = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int W = p.width, V = p.V, nt = n_tokens(V, W);
    const Layout lay = layout(W, p.max_frames);
    uint8_t* st = p.state + (long long)u * lay.bytes;
    Header* hdr = reinterpret_cast<Header*>(st);
    Beams saved = beams_at(st + lay.beams, W);
    Node* nodes = reinterpret_cast<Node*>(st + lay.nodes);
    u64* masks = reinterpret_cast<u64*>(st + lay.masks);

    int T = p.T[u] > 0 ? p.T[u] : 0;
    int frames = 0, nb = 1, cur = 0;
    long long exp2 = 0;
    double log_z = 0.0;
    const u64 tag = tag_of(V, p.blank, W, p.max_frames);
    bool refused = p.resume && hdr->tag != tag;      // not a state of such a search
    if (p.resume && !refused) {
        frames = hdr->frames;
        nb = hdr->nb;
        exp2 = hdr->exp2;
        log_z = hdr->log_z;
    }
    refused = refused || T > p.max_frames - frames;
    if (refused && tid == 0) report_error(p.err, kErrBadArgs);
    Beams b = s.b[0];
    if (tid < W && tid < nb && !refused) {
        if (p.resume) {
            b.pb[tid] = saved.pb[tid];
            b.pn[tid] = saved.pn[tid];
            b.mask[tid] = saved.mask[tid];
            b.node[tid] = saved.node[tid];
            b.last[tid] = saved.last[tid];
            b.len[tid] = saved.len[tid];
            b.pnode[tid] = saved.pnode[tid];
            b.par[tid] = saved.par[tid];
            b.head[tid] = saved.head[tid];
        } else {
            b.pb[0] = 1.0;
            b.pn[0] = 0.0;
            b.mask[0] = 0;
            b.node[0] = 0;
            b.last[0] = -1;
            b.len[0] = 0;
            b.pnode[0] = -1;
            b.par[0] = -1;
            b.head[0] = -1;
            nodes[0] = Node{-1, -1, -1, -1};
        }
    }
    for (int i = tid; i < W * s.words; i += kThreads) s.bits[i] = 0;
    if (tid < W) {
        int at = 0;
        for (int i = 0; i < tid; i++) at += pairs_of(i, V, W);
        for (int j = 0; j < pairs_of(tid, V, W); j++) s.pair[at + j] = (uint16_t)(tid << 8 | j);
    }
    __syncthreads();

    const float* row = p.logits + p.off[u] * V;
    for (int t = 0; t < (refused ? 0 : T); t++, row += V) {
        b = s.b[cur];
        Beams n = s.b[cur ^ 1];
        // the row: maximum, exp(logit - max), sum
        float mx = -INFINITY;
        for (int v = tid; v < V; v += kThreads) mx = fmaxf(mx, clean(row[v]));
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (lane == 0) red_f[warp] = mx;
        if (tid == 0) { best_key = 0; n_new = 0; n_back = 0; }
        __syncthreads();
        for (int i = 0; i < kThreads / 32; i++) mx = fmaxf(mx, red_f[i]);
        double z = 0.0;
        for (int v = tid; v < V; v += kThreads) {
            const float x = clean(row[v]);
            const double e = x == -INFINITY ? 0.0 : exp((double)x - (double)mx);
            s.p[v] = e;
            z += e;
        }
        for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        if (lane == 0) red_d[warp] = z;
        if (tid < nb && b.par[tid] >= 0)
            atomicOr(&s.bits[b.par[tid] * s.words + (b.last[tid] >> 5)], 1u << (b.last[tid] & 31));
        __syncthreads();
        z = 0.0;
        for (int i = 0; i < kThreads / 32; i++) z += red_d[i];
        if (z > 0.0) log_z += log(z);
        // tokens by probability (equal ones by id)
        for (int v = tid; v < V; v += kThreads) {
            if (v == p.blank) continue;
            const double e = s.p[v];
            int r = 0;
            for (int w = 0; w < V; w++) {
                const double f = s.p[w];
                r += w != p.blank && (f > e || (f == e && w < v));
            }
            if (r < nt) { s.stok[r] = v; s.sp[r] = e; }
        }
        __syncthreads();
        // candidates
        u64 top = 0;
        for (int c = tid; c < W + p.n_pairs; c += kThreads) {
            double val = 0.0;
            uint32_t ord = 0;
            if (c < W) {
                ord = (uint32_t)c;
                if (c < nb) {
                    double from = b.pn[c];
                    const int q = b.par[c];
                    if (q >= 0) from += b.last[q] == b.last[c] ? b.pb[q] : b.pb[q] + b.pn[q];
                    val = (b.pb[c] + b.pn[c]) * s.p[p.blank];
                    if (b.last[c] >= 0) val += from * s.p[b.last[c]];
                }
            } else {
                const int i = s.pair[c - W] >> 8, j = s.pair[c - W] & 255;
                if (i < nb) {
                    const int tok = s.stok[j];
                    ord = (uint32_t)(W + i * V + tok);
                    if (!(s.bits[i * s.words + (tok >> 5)] >> (tok & 31) & 1u))
                        val = (tok == b.last[i] ? b.pb[i] : b.pb[i] + b.pn[i]) * s.sp[j];
                }
            }
            const u64 k = (u64)__double_as_longlong(val);   // positive numbers order as their bits
            s.key[c] = k;
            s.order[c] = ord;
            top = k > top ? k : top;
        }
        atomicMax(&best_key, top);
        if (tid < W) s.slot[tid] = -1;
        __syncthreads();
        // the `width` largest, in order
        const double best = __longlong_as_double((long long)best_key);
        const u64 least = (u64)__double_as_longlong(fmax(best * 0x1p-1000, DBL_MIN));
        for (int c = tid; c < W + p.n_pairs; c += kThreads) {
            const u64 k = s.key[c];
            if (k < least) continue;
            const uint32_t o = s.order[c];
            int r = 0;
            for (int d = 0; d < W + p.n_pairs; d++) r += s.key[d] > k || (s.key[d] == k && s.order[d] < o);
            if (r < W) {
                s.sel[r] = c;
                if (c < W) s.slot[c] = r;
                atomicMax(&n_new, r + 1);
            }
        }
        if (tid < nb && b.par[tid] >= 0) s.bits[b.par[tid] * s.words + (b.last[tid] >> 5)] = 0;
        __syncthreads();
        // the new beams
        const int e2 = best > 0.0 ? ilogb(best) : 0;
        const double scale = scalbn(1.0, -e2);
        const int nn = n_new;
        int fresh = -1;          // the old beam whose new child this thread's beam is
        if (tid < nn) {
            const int c = s.sel[tid];
            if (c < W) {
                double from = b.pn[c];
                const int q = b.par[c];
                if (q >= 0) from += b.last[q] == b.last[c] ? b.pb[q] : b.pb[q] + b.pn[q];
                n.pb[tid] = (b.pb[c] + b.pn[c]) * s.p[p.blank] * scale;
                n.pn[tid] = b.last[c] >= 0 ? from * s.p[b.last[c]] * scale : 0.0;
                n.node[tid] = b.node[c];
                n.last[tid] = b.last[c];
                n.len[tid] = b.len[c];
                n.pnode[tid] = b.pnode[c];
            } else {
                const int i = s.pair[c - W] >> 8, tok = s.stok[s.pair[c - W] & 255];
                int id = -1;
                if (b.mask[i] >> (tok & 63) & 1)
                    for (id = b.head[i]; id >= 0 && nodes[id].tok != tok; id = nodes[id].next) {}
                if (id >= 0) {   // reached again after it was dropped
                    n.head[tid] = nodes[id].head;
                    n.mask[tid] = masks[id];
                    s.back[atomicAdd(&n_back, 1)] = tid;
                } else {
                    id = 1 + (frames + t) * W + tid;
                    n.head[tid] = -1;
                    n.mask[tid] = 0;
                    fresh = i;
                }
                n.pb[tid] = 0.0;
                n.pn[tid] = __longlong_as_double((long long)s.key[c]) * scale;
                n.node[tid] = id;
                n.last[tid] = tok;
                n.len[tid] = b.len[i] + 1;
                n.pnode[tid] = b.node[i];
            }
        }
        __syncthreads();
        if (fresh >= 0) {
            const int tok = n.last[tid], id = n.node[tid];
            nodes[id] = Node{b.node[fresh], tok, -1, atomicExch(&b.head[fresh], id)};
            atomicOr(&b.mask[fresh], (u64)1 << (tok & 63));
        }
        __syncthreads();
        if (tid < nb) {
            const int r = s.slot[tid];
            if (r >= 0) {
                n.head[r] = b.head[tid];
                n.mask[r] = b.mask[tid];
            } else {
                nodes[b.node[tid]].head = b.head[tid];
                masks[b.node[tid]] = b.mask[tid];
            }
        }
        if (tid < nn) {
            const int c = s.sel[tid];
            const int q = c < W ? b.par[c] : s.pair[c - W] >> 8;
            int par = q >= 0 ? s.slot[q] : -1;
            if (par < 0 && c < W)
                for (int i = 0; i < n_back; i++)
                    if (n.node[s.back[i]] == n.pnode[tid]) par = s.back[i];
            n.par[tid] = par;
        }
        exp2 += e2;
        nb = nn;
        cur ^= 1;
        __syncthreads();
    }
    b = s.b[cur];

    // state for the next call
    if (!refused) {
        if (tid == 0) {
            hdr->frames = frames + T;
            hdr->nb = nb;
            hdr->tag = tag;
            hdr->exp2 = exp2;
            hdr->log_z = log_z;
        }
        if (tid < nb) {
            saved.pb[tid] = b.pb[tid];
            saved.pn[tid] = b.pn[tid];
            saved.mask[tid] = b.mask[tid];
            saved.node[tid] = b.node[tid];
            saved.last[tid] = b.last[tid];
            saved.len[tid] = b.len[tid];
            saved.pnode[tid] = b.pnode[tid];
            saved.par[tid] = b.par[tid];
            saved.head[tid] = b.head[tid];
        }
    }
    // hypotheses, best first
    const int have = refused ? 0 : nb < p.n_best ? nb : p.n_best;
    for (int h = warp; h < p.n_best; h += kThreads / 32) {
        const long long at = (long long)u * p.n_best + h;
        const int len = h < have ? b.len[h] : -1;
        int* out = p.ids + at * p.cap;
        for (long long i = (len > 0 ? len : 0) + lane; i < p.cap; i += 32) out[i] = -1;
        if (lane) continue;
        p.n_ids[at] = len;
        p.scores[at] = h < have ? log(b.pb[h] + b.pn[h]) + (double)exp2 * 0.69314718055994530942 - log_z
                                : -INFINITY;
        if (len > 0)
            for (int i = len - 1, id = b.node[h]; i >= 0; i--, id = nodes[id].parent)
                if (i < p.cap) out[i] = nodes[id].tok;
    }
}

}  // namespace cb
}  // namespace w2v

using namespace w2v::cb;

extern "C" long long w2v_ctc_beam_state_bytes(int n_utt, int V, int width, int max_frames) {
    if (n_utt < 0 || V < 2 || V > kMaxVocab || width < 1 || width > kMaxWidth || max_frames < 1 ||
        (long long)width * max_frames >= 0x7fffffffLL)
        return -1;
    return n_utt * layout(width, max_frames).bytes;
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
    const int smem = (int)smem_layout(nullptr, nullptr, V, width, p.n_pairs);
    if (smem > 40 * 1024 &&          // beside the static part
        cudaFuncSetAttribute(ctc_beam_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return W2V_ERR_LAUNCH;
    ctc_beam_kernel<<<n_utt, kThreads, smem, reinterpret_cast<cudaStream_t>(stream)>>>(p);
    return cudaPeekAtLastError() == cudaSuccess ? W2V_OK : W2V_ERR_LAUNCH;
}
