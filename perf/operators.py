"""The operators of batched serving, as timed cases through ``Kernels``: a ragged batch of sequences
over one paged KV cache, and the token drawn from its logits.

A case is a dict of plain values. ``kind`` names the operator:

  append  Kernels.paged_append: bias, position rotation and the keys and values into their pages
  attend  Kernels.paged_attention: attention of the batch's tokens over their pages, with a sliding
          window and first tokens that stay visible (``window``, ``sinks``), or with a prefix whose
          pages all sequences share (``shared``)
  sample  Kernels.sample: temperature, top-k, top-p and min-p from given random numbers

Lengths of a batch spread over ``lo`` .. ``hi`` positions and ``nlo`` .. ``nhi`` new tokens per
sequence (one each: a decode step), the same ones for every seed. Rotary base 1e6 and head layouts
are those of this repository's model shapes; activations are N(0, 1), keys and values too, queries
twice that; logits are N(0, 2) with some peaks, as a language model's are.
"""
import math
import random

import torch

own = False

BF16 = torch.bfloat16
THETA = 1000000.0

_kernels = None


def kernels():
    global _kernels
    if _kernels is None:
        from nanoserve_amd.ops import Kernels
        _kernels = Kernels()
    return _kernels


def _batch(name, kind, b, lo, hi, nlo=1, nhi=1, heads=28, kv=4, dim=128, page=16, window=0, sinks=0,
           shared=0):
    case = {"kind": kind, "b": b, "lo": lo, "hi": hi, "nlo": nlo, "nhi": nhi, "heads": heads,
            "kv": kv, "dim": dim, "page": page, "window": window, "sinks": sinks, "shared": shared}
    return {"name": name, **case} if name else case


def listed():
    return [
        # sixteen conversations decoding together: their tokens' keys and values, the smallest append
        _batch("append decode 16", "append", 16, 100, 8000),
        # a full prompt step of several requests, some of them later chunks of long prompts
        _batch("append prompts", "append", 6, 900, 20000, 500, 900),
        # one short conversation of the 1.5B layout: the smallest attention, where latency counts
        _batch("decode 1 at 700", "attend", 1, 700, 700, heads=12, kv=2),
        # sixteen conversations of very different lengths decoding together
        _batch("decode 16 ragged", "attend", 16, 33, 8191, page=32),
        # a few very long conversations
        _batch("decode 4 at 98k", "attend", 4, 96001, 98304, page=64),
        # long conversations kept to a window of recent tokens and the first four
        _batch("decode 32 window", "attend", 32, 3000, 30000, window=4096, sinks=4),
        # the prompts of several requests, some of them behind cached tokens
        _batch("prompts ragged", "attend", 5, 2000, 8000, 301, 2000),
        # a long prompt kept to a window, of a layout with small heads
        _batch("prompt 4k window", "attend", 1, 4095, 4095, 4095, 4095, heads=14, kv=2, dim=64,
               window=1000, sinks=16),
        # a batch of short conversations behind one long system prompt
        _batch("decode 32 shared 4k", "attend", 32, 4200, 4900, shared=4096),
        # many requests over one long document, drafts of up to three tokens checked at once
        _batch("draft 96 shared 16k", "attend", 96, 16400, 17300, 1, 3, shared=16384, page=128),
        # one conversation's next token with the usual settings: the smallest draw
        {"name": "sample 1", "kind": "sample", "b": 1, "v": 152064, "type": "bf16", "rows": "same",
         "temperature": 0.7, "top_k": 20, "top_p": 0.8, "min_p": 0.0},
        # a large batch whose requests bring their own settings
        {"name": "sample 256 mixed", "kind": "sample", "b": 256, "v": 151936, "type": "fp32",
         "rows": "mixed", "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt", "shared", "shared", "sample",
                       "sample"])
    if kind == "sample":
        b = _log_int(rng, 1, 256)
        v = _log_int(rng, 1000, 152064)
        return {"kind": "sample", "b": b, "v": v, "type": rng.choice(["bf16", "fp32"]),
                "rows": rng.choice(["same", "same", "mixed"]),
                "temperature": rng.choice([0.3, 0.7, 1.0, 1.5]),
                "top_k": rng.choice([0, 0, 1, 20, 50, _log_int(rng, 2, v)]),
                "top_p": rng.choice([1.0, 0.8, 0.95, round(rng.uniform(0.05, 0.99), 3)]),
                "min_p": rng.choice([0.0, 0.0, 0.02, 0.1])}
    heads, kv, dim = rng.choice([(28, 4, 128), (12, 2, 128), (32, 8, 128), (16, 16, 128), (14, 2, 64),
                                 (40, 8, 128), (16, 16, 64), (16, 1, 128)])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    lay = dict(heads=heads, kv=kv, dim=dim, page=page)
    window, sinks = rng.choice([(0, 0), (0, 0), (_log_int(rng, 16, 8192), rng.choice([0, 1, 4, 64]))])
    if kind == "append":
        b = _log_int(rng, 1, 64)
        n = rng.choice([1, _log_int(rng, 1, 3000 // b)])
        hi = _log_int(rng, n + 1, 20000)
        return _batch(None, "append", b, rng.randrange(1, hi + 1), hi, rng.randrange(1, n + 1), n, **lay)
    if kind == "decode":
        b = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, min(98304, 1500000 // (b * kv)))
        return _batch(None, "attend", b, rng.randrange(1, hi + 1), hi, window=window, sinks=sinks, **lay)
    if kind == "prompt":
        b = _log_int(rng, 1, 8)
        n = _log_int(rng, 2, 4000 // b)
        hi = _log_int(rng, n, max(n, min(6000, 400000000 // (n * b * heads))))
        return _batch(None, "attend", b, rng.randrange(n, hi + 1), hi, rng.randrange(1, n + 1), n,
                      window=window, sinks=sinks, **lay)
    b = _log_int(rng, 2, 96)
    shared = _log_int(rng, 200, 16384)
    n = rng.choice([1, 1, 4])
    hi = shared + _log_int(rng, n, 900)
    return _batch(None, "attend", b, rng.randrange(shared + n, hi + 1), hi, 1, n, shared=shared,
                  window=window, sinks=sinks, **lay)


# ---------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case):
    """(positions, new tokens) of every sequence of a batch."""
    rng = random.Random(f"{case['b']} {case['lo']} {case['hi']} {case['nlo']} {case['nhi']}")
    new = [rng.randint(case["nlo"], case["nhi"]) for _ in range(case["b"])]
    return [max(rng.randint(case["lo"], case["hi"]), n) for n in new], new


def _pool(g, pages, kv, page, dim):
    return torch.randn(pages, kv, page, dim, generator=g, device="cuda").to(BF16)


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "sample":
        return _prepare_sample(case, g)
    lens, new = _lengths(case)
    b, ps, kv, dim = case["b"], case["page"], case["kv"], case["dim"]
    T = sum(new)
    common = case["shared"] // ps  # whole pages of the shared prefix, one copy for the batch
    width = -(-max(lens) // ps)
    counts = [max(-(-n // ps) - common, 0) for n in lens]
    total = common + sum(counts) + 1
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(b, width, dtype=torch.int32, device="cuda")
    table[:, :common] = order[:common]
    at = common
    for i, c in enumerate(counts):
        table[i, common:common + c] = order[at:at + c]
        at += c
    state = {"case": case, "table": table,
             "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
             "q_start": None, "host_lens": lens, "host_new": new,
             "k_pages": _pool(g, total, kv, ps, dim), "v_pages": _pool(g, total, kv, ps, dim)}
    if case["nhi"] > 1:
        state["q_start"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    if case["kind"] == "append":
        width = (case["heads"] + 2 * kv) * dim
        state["qkv"] = torch.randn(T, width, generator=g, device="cuda").to(BF16)
        state["bias"] = (torch.randn(width, generator=g, device="cuda") * 0.5).to(BF16)
        state["inv_freq"] = 1.0 / THETA ** (torch.arange(0, dim, 2, device="cuda").float() / dim)
    else:
        state["q"] = (torch.randn(T, case["heads"] * dim, generator=g, device="cuda") * 2).to(BF16)
        if own:
            state["work"] = kernels().paged_attention_workspace(
                T, b, case["heads"], kv, dim, table.shape[1] * ps, ragged=case["nhi"] > 1,
                shared=common * ps)
    return state


def _prepare_sample(case, g):
    b, v = case["b"], case["v"]
    x = torch.randn(b, v, generator=g, device="cuda") * 2
    hot = torch.randint(0, v, (b, 30), generator=g, device="cuda")
    x.scatter_add_(1, hot, torch.rand(b, 30, generator=g, device="cuda") * 12)
    state = {"case": case, "logits": x.to(BF16) if case["type"] == "bf16" else x,
             "u": torch.rand(b, generator=g, device="cuda")}
    for name in ("temperature", "top_k", "top_p", "min_p"):
        state[name] = case[name]
    if case["rows"] == "mixed":
        def pick(values, dtype):
            i = torch.randint(0, len(values), (b,), generator=g, device="cuda")
            return torch.tensor(values, dtype=dtype, device="cuda")[i]
        state["temperature"] = pick([0.0, 0.3, 0.7, 1.0, 1.5], torch.float32)
        state["top_k"] = pick([0, 0, 1, 20, 50, v // 3], torch.int32)
        state["top_p"] = pick([1.0, 0.8, 0.9, 0.95], torch.float32)
        state["min_p"] = pick([0.0, 0.0, 0.05], torch.float32)
    if own:
        state["work"] = kernels().sample_workspace(b, v, state["logits"].dtype)
    return state


# ---------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "sample": _own_sample}[kind](state)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[kind](state)


def _own_append(s):
    c = s["case"]
    q = kernels().paged_append(s["qkv"], s["bias"], s["inv_freq"], s["table"], s["lens"], s["k_pages"],
                               s["v_pages"], c["heads"], q_start=s["q_start"])
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_attend(s):
    c = s["case"]
    return {"out": kernels().paged_attention(
        s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], c["heads"], q_start=s["q_start"],
        shared=c["shared"] // c["page"] * c["page"], window=c["window"], sinks=c["sinks"],
        work=s["work"])}


def _own_sample(s):
    return {"token": kernels().sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"],
                                      s["min_p"], work=s["work"])}


def _positions(s):
    """(sequence, position) of every token row."""
    seq = torch.arange(s["lens"].shape[0], device="cuda")
    if s["q_start"] is None:
        return seq, s["lens"].long() - 1
    T = s["qkv"].shape[0]
    seq = torch.repeat_interleave(seq, s["q_start"].long().diff(), output_size=T)
    first = s["lens"].long() - s["q_start"].long()[1:]
    return seq, torch.arange(T, device="cuda") + first[seq]


def _plain_append(s):
    c = s["case"]
    heads, kv, dim, ps = c["heads"], c["kv"], c["dim"], c["page"]
    seq, pos = _positions(s)
    x = (s["qkv"].float() + s["bias"].float()).view(-1, heads + 2 * kv, dim)
    angle = (pos.double()[:, None] * s["inv_freq"].double())[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    lo, hi = x[:, :heads + kv, :dim // 2], x[:, :heads + kv, dim // 2:]
    rot = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(BF16)
    page = s["table"][seq, pos // ps].long()
    s["k_pages"][page, :, pos % ps] = rot[:, heads:]
    s["v_pages"][page, :, pos % ps] = x[:, heads + kv:].to(BF16)
    return {"q": rot[:, :heads].reshape(-1, heads * dim), "k_pages": s["k_pages"],
            "v_pages": s["v_pages"]}


def _plain_attend(s):
    c = s["case"]
    heads, kv, dim, ps = c["heads"], c["kv"], c["dim"], c["page"]
    rep = heads // kv
    out, row = [], 0
    for b, (n, new) in enumerate(zip(s["host_lens"], s["host_new"])):
        ids = s["table"][b, :-(-n // ps)].long()
        k, v = (p[ids].transpose(0, 1).reshape(kv, -1, dim)[:, :n].float()
                for p in (s["k_pages"], s["v_pages"]))
        q = s["q"][row:row + new].float().view(new, kv, rep, dim).permute(1, 0, 2, 3)
        score = q.reshape(kv, new * rep, dim) @ k.transpose(1, 2).contiguous() / math.sqrt(dim)
        pos = torch.arange(n - new, n, device="cuda").repeat_interleave(rep)[:, None]
        key = torch.arange(n, device="cuda")
        seen = key <= pos
        if c["window"]:
            seen &= (key > pos - c["window"]) | (key < c["sinks"])
        score = score.masked_fill(~seen, float("-inf"))
        p = (score - score.amax(-1, keepdim=True)).exp()
        o = (p / p.sum(-1, keepdim=True)) @ v
        out.append(o.view(kv, new, rep, dim).permute(1, 0, 2, 3).reshape(new, heads * dim))
        row += new
    return {"out": torch.cat(out).to(BF16)}


def _plain_sample(s):
    """Weights in 64 bits: a border that falls near a weight's edge decides the token."""
    x = s["logits"].double()
    b, v = x.shape

    def column(value, dtype):
        return torch.as_tensor(value, dtype=dtype, device="cuda").expand(b)[:, None]

    temp = column(s["temperature"], torch.float32).double()
    k = column(s["top_k"], torch.int32)
    z, order = torch.sort(x, dim=1, descending=True, stable=True)
    z = (z - z[:, :1]) / torch.where(temp > 0, temp, 1.0)
    rank = torch.arange(v, device="cuda")
    w = z.exp() * ((k <= 0) | (rank < k))
    total = w.sum(1, keepdim=True)
    before = w.cumsum(1) - w
    top_p = column(s["top_p"], torch.float32).double()
    keep = (top_p >= 1) | (before < top_p * total) | (rank == 0)
    keep &= z.exp() >= column(s["min_p"], torch.float32).double()
    keep = torch.where(temp > 0, keep, rank == 0)
    w = torch.zeros_like(x).scatter_(1, order, w * keep)
    cum = w.cumsum(1)
    hit = cum > s["u"].double()[:, None] * cum[:, -1:]
    return {"token": hit.to(torch.int8).argmax(1).to(torch.int32)}


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return {"token": torch.tensor([_exact_token(s, r) for r in range(case["b"])],
                                      dtype=torch.int32, device="cuda")}
    heads, kv, dim, ps = case["heads"], case["kv"], case["dim"], case["page"]
    lens, new = s["host_lens"], s["host_new"]
    row = 0
    if case["kind"] == "append":
        x = s["qkv"].double() + s["bias"].double()
        pools = {"k_pages": s["k_pages"].double(), "v_pages": s["v_pages"].double()}
        qs = []
        for b in range(case["b"]):
            pos = torch.arange(lens[b] - new[b], lens[b], device="cuda")
            y = x[row:row + new[b]].view(new[b], heads + 2 * kv, 2, dim // 2)
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                               torch.outer(pos.double(), s["inv_freq"].double()))[:, None]
            r = torch.complex(y[:, :heads + kv, 0], y[:, :heads + kv, 1]) * turn
            r = torch.stack([r.real, r.imag], 2).flatten(2)
            qs.append(r[:, :heads].flatten(1))
            page = s["table"][b].long()[torch.div(pos, ps, rounding_mode="floor")]
            pools["k_pages"][page, :, pos % ps] = r[:, heads:]
            pools["v_pages"][page, :, pos % ps] = y[:, heads + kv:].flatten(2)
            row += new[b]
        return {"q": torch.cat(qs), **pools}
    out = torch.zeros(sum(new), heads, dim, dtype=torch.float64, device="cuda")
    for b in range(case["b"]):
        pos = torch.arange(lens[b], device="cuda")
        page, at = s["table"][b].long()[torch.div(pos, ps, rounding_mode="floor")], pos % ps
        qpos = torch.arange(lens[b] - new[b], lens[b], device="cuda")[:, None]
        hidden = pos > qpos
        if case["window"] > 0:
            hidden = hidden | ((pos <= qpos - case["window"]) & (pos >= case["sinks"]))
        for g in range(kv):
            k, v = s["k_pages"][page, g, at].double(), s["v_pages"][page, g, at].double()
            for h in range(g * heads // kv, (g + 1) * heads // kv):
                q = s["q"][row:row + new[b], h * dim:(h + 1) * dim].double()
                p = torch.softmax((q @ k.t() * dim ** -0.5).masked_fill_(hidden, -math.inf), -1)
                out[row:row + new[b], h] = p @ v
        row += new[b]
    return {"out": out.flatten(1)}


def _exact_token(s, r):
    x = s["logits"][r].double()

    def setting(name):
        value = s[name]
        return float(value[r] if torch.is_tensor(value)
                     else torch.tensor(value, dtype=torch.float32))

    temp, k = setting("temperature"), int(setting("top_k"))
    if temp <= 0:
        return int((x == x.max()).nonzero()[0])
    weight = torch.exp((x - x.max()) / temp)
    kept = torch.argsort(-x, stable=True)
    if 0 < k < kept.numel():
        kept = kept[:k]
    if setting("top_p") < 1:
        sums = torch.cumsum(weight[kept], 0)
        enough = int(torch.searchsorted(sums, sums[-1] * setting("top_p")))
        kept = kept[:enough + 1]
    kept = kept[weight[kept] >= setting("min_p")].sort().values
    sums = torch.cumsum(weight[kept], 0)
    i = int(torch.searchsorted(sums, sums[-1] * float(s["u"][r]), right=True))
    return int(kept[min(i, kept.numel() - 1)])


# ---------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "sample":
        b, v = case["b"], case["v"]
        return {"bytes": b * v * (2 if case["type"] == "bf16" else 4) + 8 * b, "flops": 2 * b * v}
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    lens, new = _lengths(case)
    T = sum(new)
    if case["kind"] == "append":
        values = T * (heads + 2 * kv) * dim
        return {"bytes": 4 * values + 2 * (heads + 2 * kv) * dim, "flops": 4 * values}
    window, sinks = case["window"], case["sinks"] if case["window"] else 0
    common = case["shared"] // case["page"] * case["page"]
    pairs, rows, lowest = 0, 0, common
    for n, nn in zip(lens, new):
        pairs += sum(min(p + 1, window + min(sinks, max(p + 1 - window, 0))) if window else p + 1
                     for p in range(n - nn, n))
        low = max(n - nn + 1 - window, 0) if window else 0  # below it only the first tokens are seen
        first = min(sinks, low)
        rows += max(first - common, 0) + n - max(low, common)
        lowest = min(lowest, low)
    if common:  # the shared rows that any sequence sees, read once
        rows += min(sinks, lowest) + common - lowest
    return {"bytes": 4 * T * heads * dim + 4 * rows * kv * dim, "flops": 4 * pairs * heads * dim}
