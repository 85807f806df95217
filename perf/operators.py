"""Workloads of the adapter, grouped-head and beam-search operators.

A server that transcribes one batch of utterances for many languages or
customers keeps ONE set of encoder weights and, per utterance, a low-rank
adapter beside each projection and an output head of its own; the logits then
go through the prefix beam search.  The three operators:

  lora     y = epi(x W^T + bias + s_a (x A_a^T) B_a^T), a = the row's adapter
  grouped  y = epi(x W_g^T + bias_g),                    g = the row's group
  beam     CTC prefix beam search, n best hypotheses of every utterance

`own` False runs them as elementary torch operations, True through the
engine's kernels.
"""
import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
EPI = {"f16": 0, "gelu": 1, "f32": 2, "resid": 3}
# hypotheses less likely than this beside the frame's best one are dropped
PRUNE = -1000.0 * math.log(2.0)


# ── cases ───────────────────────────────────────────────────────────────────
def listed():
    return [
        # ten live microphones' streams, decoded a tenth of a second (5 frames) at a time for 2 s: the latency of a call
        dict(op="beam", name="beam 10 streams, 5 frames a call", utts=10, t_min=100, t_max=100, hop=5, vocab=32, width=8, best=1),
        # one 10 s utterance by itself
        dict(op="beam", name="beam one 10 s", utts=1, t_min=499, t_max=499, hop=0, vocab=32, width=16, best=1),
        # the engine's usual batch, ragged
        dict(op="beam", name="beam 64 x 2-10 s", utts=64, t_min=99, t_max=499, hop=0, vocab=32, width=16, best=4),
        # long recordings, a wide beam for rescoring, a larger alphabet
        dict(op="beam", name="beam 16 x 30 s wide", utts=16, t_min=1201, t_max=1499, hop=0, vocab=94, width=100, best=10),
        # one frame of each of 16 streams through a projection: the smallest product
        dict(op="lora", name="lora 16 single frames", utts=16, t_min=1, t_max=1, k=1024, n=1024, rank=16, adapters=8, weights="f16", epi="f16"),
        # one 10 s utterance, the attention's output projection onto the residual stream
        dict(op="lora", name="lora one 10 s, residual", utts=1, t_min=499, t_max=499, k=768, n=768, rank=16, adapters=4, weights="f16", epi="resid"),
        # a whole batch through the query/key/value projection
        dict(op="lora", name="lora 64 x 10 s", utts=64, t_min=499, t_max=499, k=768, n=2304, rank=16, adapters=8, weights="f16", epi="f16"),
        # the same weights as stored blocks, as the engine keeps them
        dict(op="lora", name="lora q8 64 x 2-10 s", utts=64, t_min=99, t_max=499, k=1024, n=1024, rank=16, adapters=16, weights="q8", epi="resid"),
        # feed-forward of the large encoder, ragged, larger ranks
        dict(op="lora", name="lora 48 x 5-20 s gelu", utts=48, t_min=249, t_max=999, k=1024, n=4096, rank=32, adapters=16, weights="f16", epi="gelu"),
        # output heads of 8 languages over a few short utterances
        dict(op="grouped", name="heads 8 x 0.1-1 s", utts=8, t_min=5, t_max=49, k=768, n=48, groups=8, epi="f32", sort=False),
        # output heads of a full batch, alphabets padded to 200 tokens
        dict(op="grouped", name="heads 64 x 2-20 s", utts=64, t_min=99, t_max=999, k=1024, n=200, groups=24, epi="f32", sort=False),
        # routed experts' first product: rows sorted by expert, some experts with few rows or none
        dict(op="grouped", name="experts 32 ragged", utts=32, t_min=0, t_max=1100, k=1024, n=4096, groups=32, epi="gelu", sort=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["beam", "lora", "grouped"])
    if op == "beam":
        width = _log(rng, 1, 100)
        t_max = _log(rng, 1, 1499)
        utts = max(1, min(_log(rng, 1, 64), 30000 // t_max))
        return dict(op=op, utts=utts, t_min=rng.choice([0, t_max // 4, t_max]), t_max=t_max, hop=rng.choice([0, 0, 0, max(1, t_max // 7)]),
                    vocab=_log(rng, 3, 160), width=width, best=rng.randint(1, min(width, 10)))
    t_max = _log(rng, 1, 999)
    utts = max(1, min(_log(rng, 1, 96), 30000 // t_max))
    t_min = rng.choice([0, 1, t_max // 3, t_max])
    k = 64 * _log(rng, 4, 32)
    if op == "lora":
        rank = rng.choice([8, 16, 24, 32, 64])
        return dict(op=op, utts=utts, t_min=min(t_min, t_max), t_max=t_max, k=k, n=_log(rng, 32, 512) * 8, rank=rank,
                    adapters=_log(rng, 1, 512 // rank), weights=rng.choice(["f16", "f16", "q8"]), epi=rng.choice(["f16", "gelu", "f32", "resid"]))
    n = rng.choice([_log(rng, 5, 500), 8 * _log(rng, 64, 512)])
    return dict(op=op, utts=utts, t_min=min(t_min, t_max), t_max=t_max, k=k, n=n, groups=_log(rng, 1, 32),
                epi=rng.choice(["f16", "gelu", "f32", "resid"]), sort=rng.random() < 0.5)


# ── inputs ──────────────────────────────────────────────────────────────────
def _lengths(case):
    """Frames of each utterance: of the case alone, so that every batch of it has the same shape."""
    gen = np.random.default_rng([case["utts"], case["t_min"], case["t_max"]])
    t = gen.integers(case["t_min"], case["t_max"] + 1, case["utts"])
    t[gen.integers(case["utts"])] = case["t_max"]
    if case.get("sort") and case["utts"] > 2:   # an expert with one row at most and one with none
        few = [i for i in range(case["utts"]) if i != int(t.argmax())]
        t[few[0]], t[few[-1]] = min(1, case["t_max"]), 0
    return t


def prepare(case, seed):
    gen = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(int(gen.integers(1 << 40)))

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)

    t = _lengths(case)
    m = int(t.sum())
    s = dict(case=dict(case), lens=t.tolist(), rows=m)
    s["T"] = torch.tensor(t, dtype=torch.int32, device="cuda")
    s["off"] = torch.tensor(np.concatenate([[0], np.cumsum(t)[:-1]]), dtype=torch.int64, device="cuda")
    if case["op"] == "beam":
        # a CTC head's logits: mostly blank, bursts of one token for one to three frames, and doubt between tokens
        v = case["vocab"]
        lg = normal(max(m, 1), v, std=1.5)
        burst = torch.rand(max(m, 1), device="cuda", generator=g) < 0.25
        token = torch.randint(0, v, (max(m, 1),), device="cuda", generator=g)
        lg[:, 0] += 4.0
        lg.scatter_add_(1, token[:, None], (burst * 6.0)[:, None])
        s["logits"] = lg
        return s
    k, n = case["k"], case["n"]
    s["x"] = normal(max(m, 1), k, dtype=torch.float16)[:m]
    s["resid"] = normal(max(m, 1), n, std=2.0)[:m] if case["epi"] == "resid" else None
    std = 1.0 / math.sqrt(k)
    if case["op"] == "lora":
        r, a = case["rank"], case["adapters"]
        if case["weights"] == "q8":   # blocks of 32 codes and their scale, as the engine keeps them: codes [n][k], scales [k/32][n rounded up to 8]
            ld = (n + 7) // 8 * 8
            s["codes"] = torch.randint(-127, 128, (n, k), device="cuda", generator=g, dtype=torch.int8)
            s["scales"] = (torch.rand(k // 32, ld, device="cuda", generator=g) + 0.5).mul_(std / 73.0).half()
        else:
            s["w"] = normal(n, k, std=std, dtype=torch.float16)
        s["bias"] = normal(n, std=0.1)
        s["la"] = normal(a, r, k, std=std, dtype=torch.float16)
        s["lb"] = normal(a, n, r, std=0.5 / math.sqrt(r), dtype=torch.float16)
        s["scale"] = torch.rand(a, device="cuda", generator=g) + 0.5
        pick = gen.integers(-1 if case["utts"] > 3 else 0, a, case["utts"])   # -1: an utterance without an adapter
        s["adapter"] = torch.tensor(pick, dtype=torch.int32, device="cuda")
        return s
    e = case["groups"]
    s["w"] = normal(e, n, k, std=std, dtype=torch.float16)
    s["bias"] = normal(e, n, std=0.1)
    pick = np.arange(case["utts"]) % e if case["sort"] else gen.integers(0, e, case["utts"])
    s["groups"] = (np.sort(pick) if case["sort"] else pick).tolist()
    s["group"] = torch.tensor(s["groups"], dtype=torch.int32, device="cuda")
    return s


# ── plain forms ─────────────────────────────────────────────────────────────
def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))


def _epilogue(y, case, resid):
    if case["epi"] == "gelu":
        y = _gelu(y)
    if case["epi"] == "resid":
        y = y + resid
    return y.half() if case["epi"] in ("f16", "gelu") else y


def _plain_lora(s):
    case, m = s["case"], s["rows"]
    r, a = case["rank"], case["adapters"]
    x = s["x"].float()
    if case["weights"] == "q8":   # a weight is its code times its block's scale, held in fp16
        d = s["scales"][:, : case["n"]].t().repeat_interleave(32, 1)
        w = (s["codes"].half() * d).float()
    else:
        w = s["w"].float()
    row = torch.repeat_interleave(s["adapter"], s["T"].long(), output_size=m)
    mine = (row[:, None] == torch.arange(a, device="cuda")) * s["scale"]
    t = (x @ s["la"].float().reshape(a * r, -1).t()).view(m, a, r) * mine[:, :, None]
    y = x @ w.t() + s["bias"] + t.view(m, a * r) @ s["lb"].float().transpose(1, 2).reshape(a * r, -1)
    return _epilogue(y, case, s["resid"])


def _plain_grouped(s):
    case = s["case"]
    x, w = s["x"].float(), s["w"].float()
    y = torch.cat([xs @ w[e].t() + s["bias"][e] for xs, e in zip(x.split(s["lens"]), s["groups"])])
    return _epilogue(y, case, s["resid"])


def _plain_beam(s):
    """The search on logarithms in 64 bits (scores near a cut differ by less
    than 32 bits tell apart after a thousand frames), all utterances at once,
    frame by frame; the two modular hashes of a prefix tell whether one beam
    is another's parent."""
    case = s["case"]
    b, k, v, cap = case["utts"], case["width"], case["vocab"], case["t_max"]
    neg = -math.inf
    dev = dict(device="cuda")
    p1, p2 = 2147483629, 2147483587
    pb = torch.full((b, k), neg, dtype=torch.float64, **dev)
    pb[:, 0] = 0.0
    pn = torch.full((b, k), neg, dtype=torch.float64, **dev)
    last = torch.full((b, k), -1, dtype=torch.int64, **dev)
    n = torch.zeros(b, k, dtype=torch.int64, **dev)
    h1, h2 = torch.zeros_like(n), torch.zeros_like(n)
    ids = torch.full((b, k, cap + 1), -1, dtype=torch.int32, **dev)
    tokens = torch.arange(v, **dev)
    slot = torch.arange(k, **dev)
    for t in range(cap):
        live = t < s["T"][:, None]
        row = (s["off"] + t).clamp_(max=max(s["rows"] - 1, 0))
        lp = torch.log_softmax(s["logits"][row].double(), 1)
        total = torch.logaddexp(pb, pn)
        at_last = torch.gather(lp, 1, last.clamp(min=0))
        at_last = torch.where(last >= 0, at_last, neg)
        # child[b, i, j]: beam j is beam i with beam j's last token behind it
        step = last[:, None, :] + 1
        child = ((h1[:, :, None] * 1000003 + step) % p1 == h1[:, None, :]) & ((h2[:, :, None] * 998244353 + step) % p2 == h2[:, None, :])
        child &= (n[:, :, None] + 1 == n[:, None, :]) & (total[:, :, None] > neg) & (total[:, None, :] > neg)
        grow = torch.where(last[:, :, None] == last[:, None, :], pb[:, :, None], total[:, :, None])
        from_parent = torch.where(child, grow, neg).amax(1)
        stay_b = total + lp[:, :1]
        stay_n = torch.logaddexp(pn, from_parent) + at_last
        # extensions; those that are beams already have gone into the beam
        ext = torch.where(tokens == last[:, :, None], pb[:, :, None], total[:, :, None]) + lp[:, None, :]
        ext[:, :, 0] = neg
        taken = torch.zeros(b, k, v + 1, dtype=torch.bool, **dev)
        taken.scatter_(2, torch.where(child, last[:, None, :], v), True)
        ext = torch.where(taken[:, :, :v], neg, ext)
        cand = torch.cat([torch.logaddexp(stay_b, stay_n), ext.reshape(b, k * v)], 1)
        cand = torch.where(cand < cand.amax(1, keepdim=True) + PRUNE, neg, cand)
        score, pick = torch.sort(cand, dim=1, descending=True, stable=True)
        score, pick = score[:, :k], pick[:, :k]
        stays = pick < k
        old = torch.where(stays, pick, (pick - k) // v)
        tok = torch.where(stays, 0, (pick - k) % v)
        got = score > neg

        def moved(x):
            return torch.gather(x, 1, old)

        new_n = moved(n)
        new_ids = torch.gather(ids, 1, old[:, :, None].expand(-1, -1, cap + 1))
        spot = torch.where(stays | ~got, cap, new_n)
        new_ids.scatter_(2, spot[:, :, None], tok[:, :, None].int())
        new_ids[:, :, cap] = -1
        ids = torch.where(live[:, :, None], new_ids, ids)
        nb = torch.where(got & stays, moved(stay_b), neg)
        nn = torch.where(got, torch.where(stays, moved(stay_n), score), neg)
        g1 = torch.where(stays, moved(h1), (moved(h1) * 1000003 + tok + 1) % p1)
        g2 = torch.where(stays, moved(h2), (moved(h2) * 998244353 + tok + 1) % p2)
        nl = torch.where(stays, moved(last), tok)
        new_n = new_n + (~stays).long()
        pb, pn, last = torch.where(live, nb, pb), torch.where(live, nn, pn), torch.where(live, nl, last)
        n, h1, h2 = torch.where(live, new_n, n), torch.where(live, g1, h1), torch.where(live, g2, h2)
    best = case["best"]
    score = torch.logaddexp(pb, pn)[:, :best]
    some = score > neg
    return dict(ids=torch.where(some[:, :, None], ids[:, :best, :cap], -1), n_ids=torch.where(some, n[:, :best], -1).int(), scores=score)


# ── the engine's kernels ────────────────────────────────────────────────────
def _binding():
    if "w2v_b200" not in sys.modules:
        pkg = ROOT / "wav2vec2.cpp_b200"
        spec = importlib.util.spec_from_file_location("w2v_b200", pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["w2v_b200"] = mod
        spec.loader.exec_module(mod)
    import w2v_b200.binding as binding
    return binding


def _p(t):
    return 0 if t is None else t.data_ptr()


def _own_setup(s):
    """What a server keeps from call to call: output buffers, workspace, error word, and the pointers to them."""
    case, K = s["case"], _binding().kernels
    s["K"] = K
    s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if case["op"] == "beam":
        b, best, cap = case["utts"], case["best"], case["t_max"]
        s["ids"] = torch.empty(b, best, cap, dtype=torch.int32, device="cuda")
        s["n_ids"] = torch.empty(b, best, dtype=torch.int32, device="cuda")
        s["scores"] = torch.empty(b, best, dtype=torch.float64, device="cuda")
        size = K.ctc_beam_state_bytes(b, case["vocab"], case["width"], cap)
        s["beams"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        if case["hop"]:
            # the frames of each call: every stream's next `hop` (the last call's may be fewer)
            done = range(0, cap, case["hop"])
            s["calls"] = [(s["off"] + torch.clamp(s["T"].long(), max=d), (s["T"] - d).clamp(0, case["hop"])) for d in done]
        else:
            s["calls"] = [(s["off"], s["T"])]
        return
    dtype = torch.float16 if case["epi"] in ("f16", "gelu") else torch.float32
    s["y"] = torch.empty(s["rows"], case["n"], dtype=dtype, device="cuda")
    if case["op"] == "lora":
        size = K.lora_workspace_bytes(s["rows"], case["utts"], case["rank"])
        s["work"] = torch.empty(size, dtype=torch.uint8, device="cuda")


def _own(s):
    if "K" not in s:
        _own_setup(s)
    case, K, m = s["case"], s["K"], s["rows"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "beam":
        for i, (off, T) in enumerate(s["calls"]):
            final = i + 1 == len(s["calls"])
            K.ctc_beam(_p(s["logits"]), _p(off), _p(T), case["utts"], case["vocab"], 0, case["width"], case["t_max"], i > 0, _p(s["beams"]), s["beams"].numel(),
                       case["best"] if final else 0, _p(s["ids"]), case["t_max"], _p(s["n_ids"]), _p(s["scores"]), _p(s["err"]), stream)
        return dict(ids=s["ids"], n_ids=s["n_ids"], scores=s["scores"])
    k, n, epi = case["k"], case["n"], EPI[case["epi"]]
    if case["op"] == "grouped":
        K.gemm_grouped(_p(s["x"]), k, k, m, _p(s["w"]), case["groups"], n, _p(s["y"]), n, _p(s["bias"]), _p(s["resid"]), n, epi,
                       _p(s["off"]), _p(s["T"]), _p(s["group"]), case["utts"], _p(s["err"]), stream)
        return s["y"]
    lora = (_p(s["la"]), _p(s["lb"]), _p(s["scale"]), case["adapters"], case["rank"], _p(s["off"]), _p(s["T"]), _p(s["adapter"]), case["utts"],
            _p(s["work"]), s["work"].numel())
    if case["weights"] == "q8":
        K.gemm_q_lora(_p(s["x"]), k, k, m, _p(s["codes"]), _p(s["scales"]), s["scales"].shape[1], 8, n, _p(s["y"]), n, _p(s["bias"]), _p(s["resid"]), n, epi,
                      *lora, _p(s["err"]), stream)
    else:
        K.gemm_lora(_p(s["x"]), k, k, m, _p(s["w"]), n, _p(s["y"]), n, _p(s["bias"]), _p(s["resid"]), n, epi, *lora, _p(s["err"]), stream)
    return s["y"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return _plain_beam(state) if op == "beam" else _plain_lora(state) if op == "lora" else _plain_grouped(state)


# ── work and 64-bit results ─────────────────────────────────────────────────
def work(case):
    t = _lengths(case)
    m = int(t.sum())
    if case["op"] == "beam":
        v, k = case["vocab"], case["width"]
        # logits once, hypotheses once; softmax of each row, two products and three sums per beam and the product of each beam and token
        return {"bytes": 4 * m * v + case["utts"] * case["best"] * (4 * case["t_max"] + 12), "flops": m * (4 * v + 5 * k + k * v)}
    k, n = case["k"], case["n"]
    out = (2 if case["epi"] in ("f16", "gelu") else 4) + (4 if case["epi"] == "resid" else 0)
    rows = m * (2 * k + out * n)
    if case["op"] == "lora":
        r = case["rank"]
        used = min(case["adapters"], case["utts"])   # at most
        weights = n * k * (2 if case["weights"] == "f16" else 1.0625)
        return {"bytes": rows + weights + 4 * n + used * 2 * r * (k + n), "flops": 2 * m * (k * n + r * (k + n))}
    used = min(case["groups"], case["utts"])
    return {"bytes": rows + used * (2 * n * k + 4 * n), "flops": 2 * m * k * n}


def _exact_beam(case, s):
    """The definition, an utterance at a time, on a table of prefixes."""
    best, neg = case["best"], -math.inf
    lg = s["logits"].double().cpu().numpy()
    scores = np.full((case["utts"], best), neg)
    start = 0
    for u, t in enumerate(s["lens"]):
        beams = [((), 0.0, neg)]
        for row in lg[start:start + t]:
            lp = row - (row.max() + np.log(np.exp(row - row.max()).sum()))
            new = {p: [neg, neg] for p, _, _ in beams}
            for p, b, n in beams:
                total = np.logaddexp(b, n)
                new[p][0] = np.logaddexp(new[p][0], total + lp[0])
                if p:
                    new[p][1] = np.logaddexp(new[p][1], n + lp[p[-1]])
                for c in range(1, case["vocab"]):
                    e = (b if p and c == p[-1] else total) + lp[c]
                    if e > neg:
                        q = new.setdefault(p + (c,), [neg, neg])
                        q[1] = np.logaddexp(q[1], e)
            ranked = sorted(((float(np.logaddexp(*bn)), p, bn) for p, bn in new.items()), key=lambda x: -x[0])[: case["width"]]
            beams = [(p, bn[0], bn[1]) for sc, p, bn in ranked if sc > neg and sc >= ranked[0][0] + PRUNE]
        start += t
        for i, (_, b, n) in enumerate(beams[:best]):
            scores[u, i] = np.logaddexp(b, n)
    return dict(ids=None, n_ids=None, scores=torch.from_numpy(scores))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "beam":
        if s["rows"] * case["width"] * case["vocab"] > 2_500_000:
            return None
        return _exact_beam(case, s)
    y = torch.empty(s["rows"], case["n"], dtype=torch.float64, device="cuda")
    start = 0
    if case["op"] == "lora":
        picks, scale = s["adapter"].tolist(), s["scale"].double().tolist()
        if case["weights"] == "q8":
            w = (s["codes"].view(case["n"], -1, 32).half() * s["scales"][:, : case["n"]].t()[:, :, None]).view(case["n"], -1).double()
        else:
            w = s["w"].double()
    for u, t in enumerate(s["lens"]):
        x = s["x"][start:start + t].double()
        if case["op"] == "lora":
            z = x @ w.t() + s["bias"].double()
            if picks[u] >= 0:
                z += (x @ s["la"][picks[u]].double().t()) @ s["lb"][picks[u]].double().t() * scale[picks[u]]
        else:
            z = x @ s["w"][s["groups"][u]].double().t() + s["bias"][s["groups"][u]].double()
        if case["epi"] == "gelu":
            z = z * torch.special.expit(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))   # the same curve as a logistic function
        if case["epi"] == "resid":
            z = z + s["resid"][start:start + t].double()
        y[start:start + t] = z
        start += t
    return y
