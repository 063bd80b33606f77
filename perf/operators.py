"""Performance cases of the batched decode operators: the 8-bit KV cache (append, attention) and the sampler.

A case is a dict of plain values:

  kind    "append"     one pass of a cache that takes `tokens` more tokens a sequence: rewind to where the sequences
                       stood, append, and read the touched blocks back as f32
          "attention"  `tokens` query tokens a sequence over a cache of about `length` tokens a sequence
          "sample"     one token for each of `rows` rows of `vocab` logits, from given random numbers

  seqs    sequences in the batch; `ragged`: their lengths (or token counts) differ, odd ones among them
  heads, kv_heads, head_dim, window   of the attention; the values are those of the models the library has as
          presets (tiny, 1B, 4B) and, in draw(), other head layouts that the cache takes

Inputs come from the seed alone.  exact() restates the operators in 64 bits, one sequence at a time.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

BLOCK = 64  # tokens that share a scale


def listed():
    def append(name, seqs, start, tokens, kv_heads, head_dim, ragged=False):
        return {"name": name, "kind": "append", "seqs": seqs, "start": start, "tokens": tokens, "kv_heads": kv_heads,
                "head_dim": head_dim, "ragged": ragged}

    def attention(name, seqs, length, tokens, heads, kv_heads, head_dim, window=0, ragged=False):
        return {"name": name, "kind": "attention", "seqs": seqs, "length": length, "tokens": tokens, "heads": heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "window": window, "ragged": ragged}

    def sample(name, rows, vocab, temperature, top_k, top_p, min_p, mixed=False, ties=False):
        return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "temperature": temperature,
                "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed, "ties": ties}

    return [
        # decoding: one token of one sequence goes into the 1B model's cache, mid-block; all latency
        append("append_token", 1, 101, 1, 1, 256),
        # speculative decoding: five draft tokens for each of 32 sequences of the 4B shape, after a rollback
        append("append_drafts", 32, 64, 5, 4, 256, True),
        # prompts of a batch go into the cache at once: 16 documents of up to 1907 tokens, 4B shape
        append("append_prompts", 16, 0, 1907, 4, 256, True),
        # the smallest attention there is: one token of the 1B model's local layers
        attention("attend_local", 1, 517, 1, 4, 1, 256, 512),
        # one sequence far into a long conversation, the 4B shape's global layers
        attention("attend_long", 1, 32768, 1, 8, 4, 256),
        # a serving batch: 64 ragged conversations of the 4B shape decode one token each
        attention("attend_batch", 64, 4096, 1, 8, 4, 256, 0, True),
        # verifying five draft tokens of 16 sequences, 1B shape
        attention("attend_drafts", 16, 2011, 5, 4, 1, 256, 0, True),
        # a prompt over what it just put into the cache: causal, the 4B shape's local layers
        attention("attend_prompt", 1, 1907, 1907, 8, 4, 256, 1024),
        # a chat's next token with the usual settings, the models' vocabulary
        sample("sample_chat", 1, 262144, 0.8, 40, 0.95, 0.0),
        # the same for a serving batch whose users set different rules, greedy ones among them
        sample("sample_batch", 64, 262144, 0.9, 64, 0.9, 0.05, True),
        # plain sampling at temperature 1 with nothing cut off: the whole distribution counts
        sample("sample_plain", 8, 262144, 1.0, 0, 1.0, 0.0, False, True),
        # the CPU-sized model's vocabulary
        sample("sample_small", 5, 1024, 0.7, 0, 0.9, 0.02),
    ]


def draw(rng):
    def log(a, b):
        return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))

    kind = rng.choice(["append", "append", "attention", "attention", "attention", "sample", "sample"])
    if kind == "sample":
        vocab = log(500, 262144)
        return {"kind": kind, "rows": log(1, 64), "vocab": vocab, "temperature": rng.choice([0.6, 0.8, 1.0, 1.3]),
                "top_k": rng.choice([0, 0, 20, 50, log(1, vocab)]), "top_p": rng.choice([1.0, 0.95, 0.8, 0.5]),
                "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]), "mixed": rng.random() < 0.4, "ties": rng.random() < 0.3}
    heads, kv_heads, head_dim = rng.choice([(4, 1, 256), (8, 4, 256), (4, 1, 32), (8, 8, 128), (16, 2, 128),
                                            (6, 2, 64), (8, 1, 256)])
    if kind == "append":
        seqs, tokens = log(1, 32), log(1, 1500)
        tokens = max(1, min(tokens, 20_000_000 // (seqs * kv_heads * head_dim)))
        start = rng.randrange(0, 200) if tokens <= 16 else BLOCK * rng.randrange(0, 3)
        return {"kind": kind, "seqs": seqs, "start": start, "tokens": tokens, "kv_heads": kv_heads,
                "head_dim": head_dim, "ragged": rng.random() < 0.5}
    what = rng.choice(["token", "token", "drafts", "prompt"])
    seqs = log(1, 48) if what != "prompt" else rng.choice([1, 1, 2, 3])
    most = max(64, min(20000, 180_000_000 // (seqs * kv_heads * head_dim)))
    length = log(16, most if what != "prompt" else min(most, 2500))
    tokens = {"token": 1, "drafts": rng.randrange(2, 9), "prompt": log(9, 1400)}[what]
    tokens = max(1, min(tokens, length, 10_000_000_000 // (4 * head_dim * heads * seqs * length)))
    return {"kind": kind, "seqs": seqs, "length": length, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "window": rng.choice([0, 0, 512, 1024]),
            "ragged": seqs > 1 and rng.random() < 0.6}


# ------------------------------------------------------------------ the batch of a case, on the host
def _attention_shape(case):
    """(lengths, query counts) of the sequences."""
    n, L, t = case["seqs"], case["length"], case["tokens"]
    if not case["ragged"]:
        return [L] * n, [t] * n
    # from half to one and a half of the length, odd values among them; as many queries as fit
    lens = [max(1, L // 2 + (i * 7919 + 13) % (L + 1)) for i in range(n)]
    return lens, [min(t, x) for x in lens]


def _append_shape(case):
    """(lengths before, new tokens) of the sequences.  Few new tokens start inside a block and stay in it, so that
    the pass can be repeated from the same state; more of them start at a block's beginning."""
    n, start, t = case["seqs"], case["start"], case["tokens"]
    counts = [t if not case["ragged"] else max(1, t - (i * 31) % max(1, t // 2)) for i in range(n)]
    if t <= 16:
        starts = [start // BLOCK * BLOCK + (start + 11 * i * case["ragged"]) % (BLOCK + 1 - t) for i in range(n)]
    else:
        starts = [start // BLOCK * BLOCK] * n
    return starts, counts


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * int(seed) + 29)
    return g


def _keys(g, rows, kv_heads, head_dim):
    """K rows as the norm over a head leaves them: unit variance, some channels with several times the others' size."""
    gain = 0.6 + torch.rand(kv_heads, head_dim, generator=g, device="cuda")
    gain = torch.where(torch.rand(kv_heads, head_dim, generator=g, device="cuda") < 0.03, 4.0 * gain, gain)
    return torch.randn(rows, kv_heads, head_dim, generator=g, device="cuda").mul_(gain)


def _values(g, rows, kv_heads, head_dim):
    return torch.randn(rows, kv_heads, head_dim, generator=g, device="cuda").mul_(0.5)


def _attention_inputs(case, seed):
    g = _generator(seed)
    lens, counts = _attention_shape(case)
    k = _keys(g, sum(lens), case["kv_heads"], case["head_dim"])
    v = _values(g, sum(lens), case["kv_heads"], case["head_dim"])
    q = torch.randn(sum(counts), case["heads"], case["head_dim"], generator=g, device="cuda").mul_(1.5)
    return lens, counts, q, k, v


def _append_inputs(case, seed):
    """The tokens that the sequences hold already and the new ones, sequence after sequence."""
    g = _generator(seed)
    starts, counts = _append_shape(case)
    shape = case["kv_heads"], case["head_dim"]
    old = [f(g, sum(starts), *shape) for f in (_keys, _values)]
    new = [f(g, sum(counts), *shape) for f in (_keys, _values)]
    return starts, counts, old, new


def _sample_inputs(case, seed):
    g = _generator(seed)
    rows, vocab = case["rows"], case["vocab"]
    # a broad floor and some tokens that stand out, as a model's logits have them
    logits = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.0)
    up = torch.rand(rows, vocab, generator=g, device="cuda") < min(0.5, 48 / vocab)
    logits += torch.where(up, 6.0 + 2.5 * torch.randn(rows, vocab, generator=g, device="cuda"), 0.0)
    if case["ties"]:
        logits = logits.bfloat16().float()
    u = torch.rand(rows, generator=g, device="cuda").cpu().numpy()
    p = np.zeros(rows, dtype=[("temperature", "f4"), ("top_k", "i4"), ("top_p", "f4"), ("min_p", "f4"), ("u", "f4")])
    p["temperature"], p["top_k"], p["top_p"], p["min_p"] = case["temperature"], case["top_k"], case["top_p"], case["min_p"]
    if case["mixed"]:
        at = np.arange(rows)
        p["temperature"][at % 8 == 3] = 0.0
        p["top_k"][at % 4 == 1] = 0
        p["top_p"][at % 4 == 2] = 1.0
        p["min_p"][at % 3 != 0] = 0.0
    p["u"] = u
    return logits, p


# ------------------------------------------------------------------ state
_kept = []


def _context():
    """The program's one context."""
    if not _kept:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "gemma.hs_amd"))
        import gemma_hip as gh
        _kept.extend([gh, gh.Context(0)])
    return _kept


def _quantised(x):
    """Codes (int8) and scales of x[..., blocks, BLOCK, kv_heads, head_dim], one scale a block and head."""
    a = x.abs().amax(dim=(-3, -1), keepdim=True)
    # in 64 bits, where no quotient is rounded across the middle between two codes, and the scale is a / 127 rounded once
    s = torch.clamp((a.double() / 127.0).float(), min=2.0 ** -100)
    return torch.round(x.double() / s.double()).to(torch.int8), s


def _places(lens, width):
    """Row and column in a [sequences, width] table of each token of concatenated sequences."""
    n = torch.tensor(lens)
    row = torch.repeat_interleave(torch.arange(len(lens)), n)
    col = torch.arange(int(n.sum())) - torch.repeat_interleave(torch.cumsum(n, 0) - n, n)
    return row.cuda(), col.cuda()


def prepare(case, seed):
    if case["kind"] == "sample":
        logits, p = _sample_inputs(case, seed)
        s = {"case": case, "logits": logits, "rules": p}
        if own:
            s["gh"], s["ctx"] = _context()
            s["tokens"] = torch.empty(case["rows"], dtype=torch.int32, device="cuda")
        else:  # the same rules where the plain form's tensors are
            s["on"] = {f: torch.from_numpy(np.ascontiguousarray(p[f])).cuda()[:, None] for f in p.dtype.names}
        return s

    kv_heads, hd = case["kv_heads"], case["head_dim"]
    if case["kind"] == "attention":
        lens, counts, q, k, v = _attention_inputs(case, seed)
        s = {"case": case, "q": q, "counts": np.array(counts, np.int32), "seqs": np.arange(len(lens), dtype=np.int32)}
        if own:
            gh, ctx = _context()
            s["cache"] = gh.KVCache8(ctx, len(lens), max(lens), kv_heads, hd)
            torch.cuda.synchronize()  # the cache works on its context's stream
            s["cache"].append(s["seqs"], np.array(lens, np.int32), k.data_ptr(), v.data_ptr())
            s["out"] = torch.empty_like(q)
            return s
        width = -(-max(lens) // BLOCK) * BLOCK
        at = _places(lens, width)
        for name, x in (("k", k), ("v", v)):
            rows = torch.zeros(len(lens), width, kv_heads, hd, device="cuda")
            rows[at] = x
            s[name] = _quantised(rows.view(len(lens), width // BLOCK, BLOCK, kv_heads, hd))
            del rows
        s["lens"] = torch.tensor(lens, device="cuda")
        s["n_q"] = torch.tensor(counts, device="cuda")
        s["at"] = _places(counts, max(counts))
        return s

    starts, counts, old, new = _append_inputs(case, seed)
    n = len(starts)
    s = {"case": case, "new": new}
    tails = [x % BLOCK for x in starts]
    touched = [a + b for a, b in zip(tails, counts)]
    if own:
        gh, ctx = _context()
        s["cache"] = gh.KVCache8(ctx, n, max(a + b for a, b in zip(starts, counts)), kv_heads, hd)
        s["seqs"], s["starts"], s["counts"] = (np.array(x, np.int32) for x in (range(n), starts, counts))
        s["begins"] = np.array([a // BLOCK * BLOCK for a in starts], np.int32)
        s["ends"] = s["starts"] + s["counts"]
        torch.cuda.synchronize()
        if sum(starts):
            s["cache"].append(s["seqs"], s["starts"], old[0].data_ptr(), old[1].data_ptr())
        s["out"] = [torch.empty(sum(touched), kv_heads, hd, device="cuda") for _ in range(2)]
        return s
    # the plain cache: the f32 rows of the blocks that are partly filled, and room for the codes of what is touched
    width = -(-max(touched) // BLOCK) * BLOCK
    s["shape"] = (n, width, kv_heads, hd)
    row, col = _places(starts, max(1, max(starts)))
    last = torch.tensor([a // BLOCK * BLOCK for a in starts], device="cuda")[row]
    s["tail"] = [x[col >= last] for x in old]
    s["tail_at"] = _places(tails, width)
    row, col = _places(counts, width)
    s["new_at"] = (row, col + torch.tensor(tails, device="cuda")[row])
    s["all_at"] = _places(touched, width)
    s["codes"] = [torch.zeros(n, width // BLOCK, BLOCK, kv_heads, hd, dtype=torch.int8, device="cuda") for _ in range(2)]
    s["scales"] = [torch.zeros(n, width // BLOCK, 1, kv_heads, 1, device="cuda") for _ in range(2)]
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return (_run_own if own else _run_plain)[s["case"]["kind"]](s)


def _own_append(s):
    c = s["cache"]
    c.truncate(s["seqs"], s["starts"])
    c.append(s["seqs"], s["counts"], s["new"][0].data_ptr(), s["new"][1].data_ptr())
    c.read(s["seqs"], s["begins"], s["ends"], s["out"][0].data_ptr(), s["out"][1].data_ptr())
    return s["out"]


def _own_attention(s):
    s["cache"].attention(s["seqs"], s["counts"], s["q"].data_ptr(), s["case"]["heads"], s["case"]["window"],
                         out=s["out"].data_ptr())
    return s["out"]


def _own_sample(s):
    s["gh"].sample_rows(s["ctx"], s["logits"].data_ptr(), s["case"]["vocab"], s["rules"], out=s["tokens"].data_ptr())
    return s["tokens"]


_run_own = {"append": _own_append, "attention": _own_attention, "sample": _own_sample}


def _plain_append_one(s, i):
    rows = torch.zeros(s["shape"], device="cuda")
    rows[s["tail_at"]] = s["tail"][i]
    rows[s["new_at"]] = s["new"][i]
    n, width, kv_heads, hd = s["shape"]
    codes, scales = _quantised(rows.view(n, width // BLOCK, BLOCK, kv_heads, hd))
    s["codes"][i].copy_(codes)
    s["scales"][i].copy_(scales)
    back = s["codes"][i].float() * s["scales"][i]
    return back.view(n, width, kv_heads, hd)[s["all_at"]]


def _plain_append(s):
    return [_plain_append_one(s, 0), _plain_append_one(s, 1)]


def _plain_attention(s):
    c = s["case"]
    nkv, hd, G = c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    k, v = ((codes.float() * scale).flatten(1, 2) for codes, scale in (s["k"], s["v"]))
    n, width = k.shape[:2]
    T = int(s["counts"].max())
    q = torch.zeros(n, T, c["heads"], hd, device="cuda")
    q[s["at"]] = s["q"]
    rows = q.view(n, T, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(n * nkv, T * G, hd)
    keys = k.permute(0, 2, 3, 1).reshape(n * nkv, hd, width)
    score = torch.matmul(rows, keys).view(n, nkv, T, G, width) / math.sqrt(hd)
    pos = s["lens"][:, None] - s["n_q"][:, None] + torch.arange(T, device="cuda")  # of each query
    j = torch.arange(width, device="cuda")
    seen = j <= pos[..., None]
    if c["window"]:
        seen &= j > pos[..., None] - c["window"]
    score = torch.where(seen[:, None, :, None], score, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    p = (e / e.sum(-1, keepdim=True)).view(n * nkv, T * G, width)
    values = v.permute(0, 2, 1, 3).reshape(n * nkv, width, hd)
    out = torch.matmul(p, values).view(n, nkv, T, G, hd).permute(0, 2, 1, 3, 4).reshape(n, T, c["heads"], hd)
    return out[s["at"]]


def _plain_sample(s):
    on = s["on"]
    value, token = torch.sort(s["logits"], dim=1, descending=True, stable=True)  # rank order
    vocab = value.shape[1]
    rank = torch.arange(vocab, device="cuda")
    greedy = on["temperature"] == 0
    # in 64 bits: sums over the whole vocabulary are compared with fractions of one another
    t = torch.where(greedy, 1.0, on["temperature"].double())
    w = torch.exp((value.double() - value[:, :1].double()) / t)
    k = torch.where(on["top_k"] == 0, vocab, on["top_k"])
    w = torch.where(rank < k, w, 0.0)
    mass = torch.cumsum(w, dim=1)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], dim=1)
    kept = (before < on["top_p"].double() * mass[:, -1:]) & (w >= on["min_p"].double())
    kept |= rank == 0
    total = torch.where(kept, mass, 0.0).amax(dim=1, keepdim=True)
    at = (mass <= on["u"].double() * total).sum(dim=1, keepdim=True)
    return torch.gather(token, 1, torch.where(greedy, 0, at)).squeeze(1).to(torch.int32)


_run_plain = {"append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}


# ------------------------------------------------------------------ work
def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4.0 * n + 24.0 * case["rows"], "flops": 20.0 * n}
    width = case["kv_heads"] * case["head_dim"]
    if case["kind"] == "append":
        starts, counts = _append_shape(case)
        new, touched = sum(counts), sum(a % BLOCK + b for a, b in zip(starts, counts))
        # new tokens in as f32; codes out, and back in for the read; touched tokens out as f32; both K and V
        return {"bytes": 2.0 * width * (5 * new + 5 * touched), "flops": 2.0 * width * (4 * new + touched)}
    lens, counts = _attention_shape(case)
    w, nbytes, pairs = case["window"], 0.0, 0.0
    for length, c in zip(lens, counts):
        first = length - c  # position of the first query
        nbytes += length - (max(0, first - w + 1) if w else 0)
        at = np.arange(first, length, dtype=np.float64) + 1
        pairs += float((np.minimum(at, w) if w else at).sum())
    return {"bytes": nbytes * (2.0 * width + 8.0 * case["kv_heads"] / BLOCK) + 8.0 * sum(counts) * case["heads"] * case["head_dim"],
            "flops": 4.0 * case["head_dim"] * case["heads"] * pairs}


# ------------------------------------------------------------------ the same in 64 bits, from the definition
def _exact_blocks(x):
    """What a cache holds of the tokens x[tokens, kv_heads, head_dim] that begin at a block's beginning."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for i in range(0, x.shape[0], BLOCK):
        for h in range(x.shape[1]):
            b = x[i:i + BLOCK, h].double()
            scale = max(float((b.abs().max() / 127.0).float()), 2.0 ** -100)
            out[i:i + BLOCK, h] = torch.round(b / scale) * scale
    return out


def exact(case, seed):
    if case["kind"] == "sample":
        return None
    if case["kind"] == "append":
        starts, counts, old, new = _append_inputs(case, seed)
        if sum(a + b for a, b in zip(starts, counts)) * case["kv_heads"] > 500_000:
            return None
        outs = []
        for o, x in zip(old, new):
            parts, i, j = [], 0, 0
            for a, b in zip(starts, counts):
                held = torch.cat([o[i:i + a], x[j:j + b]])
                parts.append(_exact_blocks(held[a // BLOCK * BLOCK:]))
                i, j = i + a, j + b
            outs.append(torch.cat(parts))
        return outs
    lens, counts, q, k, v = _attention_inputs(case, seed)
    if sum(lens) * case["kv_heads"] > 2_000_000:
        return None
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    i = j = 0
    for length, c in zip(lens, counts):
        kd, vd = _exact_blocks(k[i:i + length]), _exact_blocks(v[i:i + length])
        at = torch.arange(length - c, length, device=q.device)[:, None]
        key = torch.arange(length, device=q.device)[None, :]
        hidden = (key > at) | ((key <= at - case["window"]) if case["window"] else False)
        for h in range(case["heads"]):
            logit = q[j:j + c, h].double() @ kd[:, h // group].T.contiguous() / math.sqrt(case["head_dim"])
            p = torch.softmax(logit.masked_fill(hidden, -math.inf), dim=1)
            out[j:j + c, h] = p @ vd[:, h // group].contiguous()
        i, j = i + length, j + c
    return out
