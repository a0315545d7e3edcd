"""Operators of a server with many requests, each with its own adapter and its own way of drawing the next token.

`adapters`: low-rank adapters of many requests at once, beside a projection that all of them share.  Row n of x belongs to adapter a = index[n]
(none where it is negative): out[n] = base[n] + scale[a] B[a] (A[a] x[n]), with A[a] the first rank[a] rows of [most, K] and B[a] the first
rank[a] columns of [M, most]; base is what the shared projection gave.

`draw`: one token per row of logits from a given random number u, after temperature, top-k, top-p and min-p.  With w_i = exp((l_i - max) / T),
and 0 for less than 2^-40: the k largest logits are kept (ties: the lower index), of these in falling order those before which the share of w is
under top_p, of these the ones with w > 0 and w >= min_p; the token is the first kept one, in vocabulary order, whose running sum of w exceeds u times the sum of
all kept.  T = 0 takes the largest logit.  The second output is the token's log-probability among the kept ones.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # One user's token with an adapter on a square projection of the 3B shape: the smallest call.
        {"name": "adapter, one session", "op": "adapters", "rows": 1, "K": 2560, "M": 2560, "adapters": 4, "rank": 16, "mixed": False, "none": False, "x": "float32", "w": "float16"},
        # The ordinary serving batch, every session with an adapter of its own, ranks of 4 to 16, behind ffn.value.
        {"name": "adapters, 64 sessions", "op": "adapters", "rows": 64, "K": 10240, "M": 2560, "adapters": 64, "rank": 16, "mixed": True, "none": False, "x": "float32", "w": "float16"},
        # The largest batch of the decode sweep on a handful of popular adapters; an eighth of the sessions has none.
        {"name": "adapters, 1024 sessions", "op": "adapters", "rows": 1024, "K": 2560, "M": 2560, "adapters": 8, "rank": 32, "mixed": False, "none": True, "x": "float32", "w": "bfloat16"},
        # A packed step of prompt chunks, before ffn.key.
        {"name": "adapters, prompt chunk", "op": "adapters", "rows": 512, "K": 2560, "M": 10240, "adapters": 3, "rank": 64, "mixed": False, "none": False, "x": "float32", "w": "float16"},
        # Prompts of many requests at once with activations of 16 bits: the largest call.
        {"name": "adapters, 4096 rows", "op": "adapters", "rows": 4096, "K": 2560, "M": 10240, "adapters": 16, "rank": 64, "mixed": True, "none": False, "x": "bfloat16", "w": "bfloat16"},
        # Sizes that are no multiple of anything.
        {"name": "adapters, odd sizes", "op": "adapters", "rows": 37, "K": 1001, "M": 777, "adapters": 5, "rank": 13, "mixed": True, "none": True, "x": "float16", "w": "float16"},
        # One user's next token with the usual chat settings.
        {"name": "draw, one session", "op": "draw", "rows": 1, "V": 65536, "how": "chat", "masked": False, "x": "float32"},
        # A few sessions of the tiny model, nucleus sampling.
        {"name": "draw, tiny", "op": "draw", "rows": 3, "V": 4096, "how": "nucleus", "masked": False, "x": "float32"},
        # The ordinary serving batch.
        {"name": "draw, 64 sessions", "op": "draw", "rows": 64, "V": 65536, "how": "chat", "masked": False, "x": "float32"},
        # The largest batch of the decode sweep, top-p over the whole vocabulary.
        {"name": "draw, 1024 sessions", "op": "draw", "rows": 1024, "V": 65536, "how": "nucleus", "masked": False, "x": "float32"},
        # Requests that each bring their own settings (greedy ones among them), some tokens forbidden.
        {"name": "draw, mixed settings", "op": "draw", "rows": 200, "V": 65536, "how": "mixed", "masked": True, "x": "float32"},
        # An odd vocabulary in 16 bits, where many logits are equal.
        {"name": "draw, odd vocabulary", "op": "draw", "rows": 256, "V": 50003, "how": "min-p", "masked": False, "x": "float16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        c = {"op": "draw", "rows": _log_int(rng, 1, 1024), "V": _log_int(rng, 500, 131072), "how": rng.choice(["chat", "nucleus", "min-p", "plain", "greedy", "mixed"]),
             "masked": rng.random() < 0.3, "x": rng.choice(["float32", "float32", "float16", "bfloat16"])}
        c["rows"] = max(1, min(c["rows"], (1 << 26) // c["V"]))
        if rng.random() < 0.5:
            c["V"] = max(8, c["V"] // 8 * 8)
        return c
    c = {"op": "adapters", "rows": _log_int(rng, 1, 4096), "K": _log_int(rng, 64, 16384), "M": _log_int(rng, 64, 16384), "adapters": _log_int(rng, 1, 128),
         "rank": _log_int(rng, 1, 128), "mixed": rng.random() < 0.5, "none": rng.random() < 0.3, "x": rng.choice(["float32", "float32", "float16", "bfloat16"])}
    c["w"] = c["x"] if c["x"] != "float32" else rng.choice(["float16", "bfloat16"])
    if rng.random() < 0.7:
        c["K"], c["M"], c["rank"] = (max(n, v // n * n) for v, n in ((c["K"], 64), (c["M"], 64), (c["rank"], 4)))
    # no more than the largest listed case costs
    c["rows"] = max(1, min(c["rows"], 4096 * (2560 + 2 * 10240) // (c["K"] + 2 * c["M"]) // (2 if c["x"] == "float32" else 1)))
    c["adapters"] = max(1, min(c["adapters"], (1 << 25) // (c["rank"] * (c["K"] + c["M"]))))
    c["rank"] = max(1, min(c["rank"], 4096 * 64 * 12800 // (c["rows"] * (c["K"] + c["M"]))))
    return c


def _ranks(c):
    """Rank of every adapter: all alike, or a full, a half and a quarter one in turn."""
    return [max(1, c["rank"] >> (a % 3)) if c["mixed"] else c["rank"] for a in range(c["adapters"])]


def _row_adapters(c):
    """Adapter of every row before they are shuffled: each in turn, and -1 for every eighth row where some have none."""
    return [-1 if c["none"] and n % 8 == 7 else n % c["adapters"] for n in range(c["rows"])]


SETTINGS = {"chat": (0.8, 50, 0.9, 0.0), "nucleus": (1.0, 0, 0.9, 0.0), "min-p": (1.2, 0, 1.0, 0.05), "plain": (1.0, 0, 1.0, 0.0), "greedy": (0.0, 0, 1.0, 0.0)}
MIXED = [SETTINGS[h] for h in ("chat", "nucleus", "min-p", "plain", "greedy")] + [(0.7, 20, 0.8, 0.02), (1.0, 1000, 0.95, 0.0), (1.5, 200, 1.0, 0.1)]


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[c["x"]]
    if c["op"] == "draw":
        R, V = c["rows"], c["V"]
        l = torch.randn(R, V, generator=g, device=dev) * 2.5
        # a few tokens of every row fit the text, in some rows one far better than all others
        fits = torch.randint(0, V, (R, 12), generator=g, device=dev)
        l.scatter_add_(1, fits, torch.rand(R, 12, generator=g, device=dev) * torch.linspace(2.0, 14.0, R, device=dev)[:, None])
        if c["masked"]:
            l.masked_fill_(torch.rand(R, V, generator=g, device=dev) < 0.05, float("-inf"))
        rows = (MIXED * (R // len(MIXED) + 1))[:R] if c["how"] == "mixed" else [SETTINGS[c["how"]]] * R
        T, k, p, m = zip(*rows)
        params = torch.empty(R, 4, device=dev)
        params[:, 0] = torch.tensor(T, device=dev)
        params[:, 1] = torch.tensor(k, dtype=torch.int32, device=dev).view(torch.float32)
        params[:, 2] = torch.tensor(p, device=dev)
        params[:, 3] = torch.tensor(m, device=dev)
        s = {"op": "draw", "logits": l.to(dt), "params": params, "u": torch.rand(R, generator=g, device=dev), "token": torch.empty(R, dtype=torch.int32, device=dev),
             "logprob": torch.empty(R, device=dev)}
        if own:
            import rwkv_rsv_b200 as rsv
            s["draw"] = rsv.draw_tokens
        return s
    R, K, M, n, most = c["rows"], c["K"], c["M"], c["adapters"], c["rank"]
    wt = DTYPES[c["w"]]
    s = {"op": "adapters", "x": torch.randn(R, K, generator=g, device=dev).to(dt), "base": torch.randn(R, M, generator=g, device=dev).to(dt), "out": torch.empty(R, M, dtype=dt, device=dev),
         "A": (torch.randn(n, most, K, generator=g, device=dev) / math.sqrt(K)).to(wt), "B": (torch.randn(n, M, most, generator=g, device=dev) * 0.2).to(wt),
         "rank": torch.tensor(_ranks(c), dtype=torch.int32, device=dev), "scale": torch.rand(n, generator=g, device=dev) + 0.5,
         "index": torch.tensor(_row_adapters(c), dtype=torch.int32, device=dev)[torch.randperm(R, generator=g, device=dev)]}
    if own:
        import rwkv_rsv_b200 as rsv
        s["adapters"] = rsv.Adapters(s["A"], s["B"], ranks=s["rank"], scales=s["scale"])
    return s


def _draw_plain(s):
    T, k, p, m = s["params"][:, 0:1].double(), s["params"][:, 1:2].view(torch.int32), s["params"][:, 2:3].double(), s["params"][:, 3:4].double()
    V = s["logits"].shape[1]
    l, at = torch.sort(s["logits"], dim=1, descending=True, stable=True)  # equal logits stay in the order of their indices
    l = l.double()  # borders between two tokens are nearer to each other than 32 bits tell apart
    w = torch.exp((l - l[:, :1]) / torch.where(T > 0, T, 1.0))
    w = torch.where(w >= 2.0**-40, w, 0.0)
    place = torch.arange(V, device=l.device)[None, :]
    keep = (place < torch.where(k > 0, k, V)) & (w >= torch.clamp(m, 2.0**-40, 1.0))
    of_k = torch.where(place < torch.where(k > 0, k, V), w, 0.0)
    upto = torch.cumsum(of_k, 1)
    keep &= (upto - of_k < p * upto[:, -1:]) | (p <= 0) | (p >= 1)
    keep &= (T > 0) | (place == 0)
    kept = torch.zeros_like(w).scatter_(1, at, torch.where(keep, w, 0.0))
    sums = torch.cumsum(kept, 1)
    total = sums[:, -1:]
    token = (sums > s["u"][:, None].double() * total).to(torch.int32).argmax(1, keepdim=True)
    return {"token": token[:, 0].to(torch.int32), "logprob": torch.log(torch.gather(kept, 1, token) / total)[:, 0].float()}


def _adapters_plain(s):
    n, most, K = s["A"].shape
    of = torch.arange(n, device=s["A"].device).repeat_interleave(most)  # adapter of every column of t
    col = torch.arange(most, device=s["A"].device).repeat(n)
    t = s["x"].float() @ s["A"].float().reshape(n * most, K).T
    t = torch.where((s["index"][:, None] == of[None, :]) & (col < s["rank"][of])[None, :], t * s["scale"][of], 0.0)
    return (s["base"].float() + t @ s["B"].float().transpose(1, 2).reshape(n * most, -1)).to(s["x"].dtype)


def run(state):
    s = state
    if own:
        if s["op"] == "draw":
            s["draw"](s["logits"], s["params"], s["u"], s["token"], s["logprob"])
            return {"token": s["token"], "logprob": s["logprob"]}
        s["adapters"].apply(s["x"], s["index"], s["out"], base=s["base"])
        return s["out"]
    return _draw_plain(s) if s["op"] == "draw" else _adapters_plain(s)


def work(case):
    c = case
    size = 4 if c["x"] == "float32" else 2
    if c["op"] == "draw":  # a difference, a scale, an exponential and an addition for every logit
        return {"bytes": c["rows"] * (c["V"] * size + 28), "flops": 4 * c["rows"] * c["V"]}
    ranks, rows = _ranks(c), _row_adapters(c)
    used = set(rows) - {-1}
    return {"bytes": sum(c["K"] * size for a in rows if a >= 0) + c["rows"] * (2 * c["M"] * size + 4) + sum(ranks[a] * (c["K"] + c["M"]) * 2 + 8 for a in used),
            "flops": sum(2 * ranks[a] * (c["K"] + c["M"]) for a in rows if a >= 0) + 2 * c["rows"] * c["M"]}


def exact(case, seed):
    """From the definitions, in 64 bits: adapter by adapter, and token by token in falling order of the logits."""
    s = prepare(case, seed)
    if s["op"] == "adapters":
        out = s["base"].double()
        index, ranks = s["index"].tolist(), s["rank"].tolist()
        for a, r in enumerate(ranks):
            rows = torch.tensor([n for n, i in enumerate(index) if i == a], dtype=torch.int64, device="cuda")
            low = torch.einsum("nk,rk->nr", s["x"][rows].double(), s["A"][a, :r].double())
            out[rows] += s["scale"][a].double() * torch.einsum("nr,mr->nm", low, s["B"][a, :, :r].double())
        return out
    token, logprob = [], []
    for n, (l, u) in enumerate(zip(s["logits"], s["u"].double().tolist())):
        T, p, m = (float(s["params"][n, i]) for i in (0, 2, 3))
        k = int(s["params"][n, 1:2].view(torch.int32)) or len(l)
        fall = torch.argsort(-l.double(), stable=True)[: 1 if T == 0 else k]
        z = (l[fall].double() - l[fall[0]].double()) / (T or 1.0)
        fall, z = fall[z >= -40 * math.log(2)], z[z >= -40 * math.log(2)]
        if m > 0:
            fall = fall[z >= math.log(m)]
        if 0 < p < 1:
            share = torch.cumsum(torch.softmax(z, 0), 0)
            fall = fall[: 1 + int((share < p).sum())]
        fall = torch.sort(fall).values
        z = (l[fall].double() - l.max().double()) / (T or 1.0)
        lp = z - torch.logsumexp(z, 0)
        hit = min(int((torch.cumsum(torch.exp(lp), 0) <= u).sum()), len(fall) - 1)
        token.append(int(fall[hit]))
        logprob.append(float(lp[hit]))
    return {"token": torch.tensor(token, dtype=torch.int32), "logprob": torch.tensor(logprob, dtype=torch.float64)}
