"""The operators at both ends of a GPT's training step, and its dropout, as training and generation call them.

A case names its operator (`op`), its sizes, its type and whether the pass is a training step
(`train`: the operator, then its gradients) or an evaluation.

ops: "embedding"   y_t = scale W[id_t] + P[position_t] of ids [batch, tokens] with the frequencies of a text's
                   tokens. `positions`: rows of the table P (0: none); `given` positions are an input, else
                   every sequence counts from 0. `padding`: the share of padded tokens, whose id takes no gradient
     "dropout"     y = dropout(x, p, seed)
     "norm"        (y, h) = dropout_add_layer_norm(x, residual, weight, bias, p, seed): h = residual + dropout(x)
                   is the residual stream as it is kept, y = layer norm of h
     "policy"      (loss, gradient of the logits, log-probabilities of the actions): the clipped policy loss with
                   a KL term against a reference model (`kl` 0: none), the mean over the tokens that count
     "preference"  (loss, gradient of the logits, log-probabilities of the sequences): the preference loss of
                   `pairs` of sequences [2 pairs, tokens, vocab], chosen ones first, of several lengths

An element of row r and column c is dropped iff its 16-bit number is below round(65536 p): number c mod 8 of the
128 bits (lower half of a word first) that Philox4x32-10 makes of counter {r ceil(dim / 8) + c // 8, seed[1]}
and key seed[0], 64-bit numbers with the lower word first.

Types: `dtype` is the tables', x's and the logits'; `stream` the residual stream's, its norm's output's and its
weights' (a 16-bit branch joins a 32-bit stream under autocast).
"""

import math
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.getcwd(), "isa-_amd"))

own = False

EPS = 1e-5
IGNORED = -100


def _embedding(name, batch, tokens, vocab, dim, dtype="float32", positions=0, given=False, scale=1.0, padding=0.0,
               train=True):
    c = {"op": "embedding", "batch": batch, "tokens": tokens, "vocab": vocab, "dim": dim, "dtype": dtype,
         "positions": positions, "given": given, "scale": scale, "padding": padding, "train": train}
    return {"name": name, **c} if name else c


def _dropout(name, rows, dim, dtype, p=0.1):
    c = {"op": "dropout", "rows": rows, "dim": dim, "dtype": dtype, "p": p, "train": True}
    return {"name": name, **c} if name else c


def _norm(name, rows, dim, dtype, stream=None, p=0.1):
    c = {"op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "stream": stream or dtype, "p": p, "train": True}
    return {"name": name, **c} if name else c


def _policy(name, rows, vocab, dtype, kl=0.04, low=0.2, high=0.2):
    c = {"op": "policy", "rows": rows, "vocab": vocab, "dtype": dtype, "kl": kl, "low": low, "high": high, "train": True}
    return {"name": name, **c} if name else c


def _preference(name, pairs, tokens, vocab, dtype, beta=0.1):
    c = {"op": "preference", "pairs": pairs, "tokens": tokens, "vocab": vocab, "dtype": dtype, "beta": beta, "train": True}
    return {"name": name, **c} if name else c


def listed():
    return [
        # generation with a GPT-L: one token at its place in a sequence; launches and latency
        _embedding("embed_token", 1, 1, 50304, 768, positions=1024, given=True, train=False),
        # fine-tuning on padded sequences of several lengths, sizes that no vector load divides, a scaled table
        _embedding("embed_ragged_step", 3, 333, 5003, 390, "bfloat16", scale=19.75, padding=0.2),
        # GPT-L training, 8 x 1024 tokens
        _embedding("embed_gptl_step", 8, 1024, 50304, 768, positions=1024),
        # training on long sequences: frequent tokens appear thousands of times
        _embedding("embed_long_step", 4, 16384, 50304, 1024, "bfloat16", scale=32.0),
        # dropout of a small batch's embeddings, odd sizes
        _dropout("dropout_ragged_step", 999, 390, "float16"),
        # dropout of a GPT-L's embeddings, 8 x 1024 tokens
        _dropout("dropout_gptl_step", 8 * 1024, 768, "float32"),
        # ViT-M training under autocast: 128 images of 65 tokens, a bf16 branch joins an fp32 stream
        _norm("drop_norm_vitm_step", 128 * 65, 256, "bfloat16", "float32"),
        # GPT-L training, 8 x 1024 tokens
        _norm("drop_norm_gptl_step", 8 * 1024, 768, "float32", p=0.2),
        # a small vocabulary, odd sizes, 16-bit logits, no reference model
        _policy("policy_small", 1023, 5003, "bfloat16", kl=0.0, high=0.28),
        # tuning a GPT-L by rewards, 8 x 1024 tokens
        _policy("policy_gptl", 8 * 1024, 50304, "float32"),
        # a few short pairs, a small vocabulary, 16-bit logits
        _preference("preference_small", 3, 171, 5003, "float16"),
        # tuning a GPT-L on pairs of sequences of up to 1024 tokens
        _preference("preference_gptl", 4, 1024, 50304, "float32"),
    ]


LARGEST = 3.4e9  # of _cost: about that of the largest listed case


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        op = rng.choice(["embedding", "embedding", "dropout", "norm", "policy", "preference"])
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        width = rng.choice([192, 256, 384, 768, size(32, 4096), 8 * size(8, 512)])
        p = rng.choice([0.1, 0.1, 0.2, 0.5, round(rng.uniform(0.01, 0.9), 3)])
        vocab = rng.choice([50304, size(100, 131072)])
        if op == "embedding":
            batch, tokens = size(1, 64), size(1, 16384)
            if batch * tokens > 131072:
                continue
            positions = rng.choice([0, tokens, tokens + size(1, 4096)])
            train = rng.random() < 0.8
            c = _embedding(None, batch, tokens, vocab, width, dtype, positions, positions > 0 and rng.random() < 0.5,
                           rng.choice([1.0, 1.0, round(math.sqrt(width), 3)]), rng.choice([0.0, 0.0, 0.1, 0.7]), train)
        elif op == "dropout":
            c = _dropout(None, size(1, 65536), width, dtype, p)
        elif op == "norm":
            c = _norm(None, size(1, 65536), width, dtype, "float32" if rng.random() < 0.4 else dtype, p)
        elif op == "policy":
            c = _policy(None, size(1, 16384), vocab, dtype, rng.choice([0.0, 0.04, 0.001, 0.2]), rng.choice([0.1, 0.2]),
                        rng.choice([0.1, 0.2, 0.28]))
        else:
            c = _preference(None, size(1, 32), size(1, 2048), vocab, dtype, rng.choice([0.05, 0.1, 0.5]))
        if _cost(c) <= LARGEST:
            return c


# ---------------------------------------------------------------------------------------
# inputs


def _text(n, vocab, g):
    """Tokens with a text's frequencies, about as 1 over their rank, at places all over the table."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.pow(vocab + 1.0, u) - 1.0).long().clamp_(0, vocab - 1)
    return torch.randperm(vocab, generator=g, device="cuda")[rank]


def _logits(rows, vocab, targets, dtype, g):
    """Logits of a model that has learnt something: the token that came stands out."""
    x = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.0)
    x.scatter_add_(1, targets[:, None], torch.full((rows, 1), 6.0, device="cuda"))
    return x.to(dtype)


def _taken(logits, targets):
    """Log-probabilities of the targets, some rows at a time."""
    return torch.cat([torch.log_softmax(x.float(), -1).gather(1, t[:, None])[:, 0]
                      for x, t in zip(logits.split(1024), targets.split(1024))])


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, c["dtype"])

    def randn(*shape, scale=1.0, to=dtype):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(to)

    s = {"case": c}
    if c["op"] == "embedding":
        b, n, v, d = c["batch"], c["tokens"], c["vocab"], c["dim"]
        ids = _text(b * n, v, g).view(b, n)
        s["padding"] = None
        if c["padding"]:  # behind sequences of several lengths
            s["padding"] = 0
            kept = torch.rand(b, 1, generator=g, device="cuda").mul_(-2.0 * c["padding"]).add_(1.0).clamp_(0.0, 1.0)
            ids = ids.masked_fill(torch.arange(n, device="cuda") >= (kept * n).ceil(), 0)
        s["ids"] = ids
        s["weight"] = randn(v, d, scale=0.02)
        if c["positions"]:
            s["position_weight"] = randn(c["positions"], d, scale=0.02)
            if c["given"]:  # sequences that go on from somewhere
                first = torch.randint(0, c["positions"] - n + 1, (b, 1), generator=g, device="cuda")
                s["positions"] = first + torch.arange(n, device="cuda")
        if c["train"]:
            s["dy"] = randn(b, n, d)
        names = ("weight", "position_weight")
    elif c["op"] in ("dropout", "norm"):
        m, d = c["rows"], c["dim"]
        s["seed"] = torch.randint(-(2 ** 62), 2 ** 62, (2,), generator=g, device="cuda")
        s["x"] = randn(m, d)
        s["dy"] = randn(m, d, to=getattr(torch, c.get("stream", c["dtype"])))
        if c["op"] == "norm":
            stream = s["dy"].dtype
            # a residual stream has channels far from zero and a few wide ones
            wide = 1.0 + 8.0 * (torch.rand(d, generator=g, device="cuda") > 0.99)
            s["residual"] = (randn(m, d, to=torch.float32) * wide + randn(d, scale=0.5, to=torch.float32)).to(stream)
            s["weight"] = (1.0 + randn(d, scale=0.2, to=torch.float32)).to(stream)
            s["bias"] = randn(d, scale=0.1, to=stream)
            s["dh"] = randn(m, d, to=stream)  # from the blocks above, past the norm
        names = ("x", "residual", "weight", "bias")
    elif c["op"] == "policy":
        m, v = c["rows"], c["vocab"]
        s["actions"] = torch.randint(0, v, (m,), generator=g, device="cuda")
        s["logits"] = _logits(m, v, s["actions"], dtype, g)
        now = _taken(s["logits"], s["actions"])
        # some steps after the samples were drawn: most ratios within the bounds, some past them. A ratio nearer to
        # a bound than the rounding of its log-probability may be taken as on either side: none is
        moved = randn(m, scale=0.15, to=torch.float32)
        for border in (math.log(1.0 - c["low"]), math.log(1.0 + c["high"])):
            moved = torch.where((moved - border).abs() < 2e-4, moved + 5e-4, moved)
        s["old"] = now - moved
        s["advantages"] = randn(m, to=torch.float32)
        s["ref"] = now - randn(m, scale=0.3, to=torch.float32) if c["kl"] else None
        # prompts and padding do not count; the first token always does
        ignored = torch.rand(m, generator=g, device="cuda") < 0.25
        ignored[:1] = False
        s["actions"].masked_fill_(ignored, IGNORED)
        names = ()
    else:
        b, n, v = 2 * c["pairs"], c["tokens"], c["vocab"]
        t = torch.randint(0, v, (b * n,), generator=g, device="cuda")
        logits = _logits(b * n, v, t, dtype, g)
        # answers of several lengths behind their prompts: one token at least counts
        prompt = (torch.rand(b, 1, generator=g, device="cuda") * 0.4 * n).floor()
        end = (prompt + 1 + torch.rand(b, 1, generator=g, device="cuda") * (n - prompt)).floor()
        at = torch.arange(n, device="cuda")
        counted = (at >= prompt) & (at < end)
        taken = (_taken(logits, t).double().view(b, n) * counted).sum(1)
        s["targets"] = t.view(b, n).masked_fill(~counted, IGNORED)
        s["logits"] = logits.view(b, n, v)
        s["ref"] = (taken + randn(b, scale=4.0, to=torch.float64)).float()
        names = ()
    if c["train"]:
        for name in names:
            if name in s:
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------
# a pass: the framework's operators


def _own_embedding(s):
    from isa.kernels.transformer_block import embedding

    c, w, p = s["case"], s["weight"], s.get("position_weight")
    how = {"scale": c["scale"], "position_weight": p, "positions": s.get("positions"), "padding_index": s["padding"]}
    if not c["train"]:
        with torch.no_grad():
            return {"y": embedding(s["ids"], w, **how)}
    y = embedding(s["ids"], w, **how)
    if p is None:
        return {"y": y.detach(), "dweight": torch.autograd.grad(y, w, s["dy"])[0]}
    dw, dp = torch.autograd.grad(y, (w, p), s["dy"])
    return {"y": y.detach(), "dweight": dw, "dposition_weight": dp}


def _own_dropout(s):
    from isa.kernels.transformer_block import dropout

    y = dropout(s["x"], s["case"]["p"], s["seed"])
    return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}


def _own_norm(s):
    from isa.kernels.transformer_block import dropout_add_layer_norm

    inputs = (s["x"], s["residual"], s["weight"], s["bias"])
    y, h = dropout_add_layer_norm(*inputs, EPS, p=s["case"]["p"], seed=s["seed"])
    dx, dr, dw, db = torch.autograd.grad((y, h), inputs, (s["dy"], s["dh"]))
    return {"y": y.detach(), "h": h.detach(), "dx": dx, "dresidual": dr, "dweight": dw, "dbias": db}


def _own_policy(s):
    from isa.kernels.transformer_block import policy_loss_with_grad

    c = s["case"]
    loss, dlogits, logp = policy_loss_with_grad(s["logits"], s["actions"], s["old"], s["advantages"], ref_logp=s["ref"],
                                                clip=(c["low"], c["high"]), kl=c["kl"], ignore_index=IGNORED)
    return {"loss": loss, "dlogits": dlogits, "logp": logp}


def _own_preference(s):
    from isa.kernels.transformer_block import preference_loss_with_grad

    loss, dlogits, logp = preference_loss_with_grad(s["logits"], s["targets"], s["ref"], beta=s["case"]["beta"],
                                                    ignore_index=IGNORED)
    return {"loss": loss, "dlogits": dlogits, "logp": logp}


# ---------------------------------------------------------------------------------------
# a pass: elementary operations in 32 bits


def _plain_embedding(s):
    c, w, ids = s["case"], s["weight"], s["ids"]
    y = w[ids].float() * c["scale"]
    at = None
    if "position_weight" in s:
        at = s["positions"] if "positions" in s else torch.arange(c["tokens"], device=ids.device).expand(ids.shape)
        y = y + s["position_weight"][at].float()
    got = {"y": y.to(w.dtype)}
    if c["train"]:
        dy = s["dy"].float().view(-1, c["dim"])
        keys = ids.reshape(-1)
        dw = torch.zeros(w.shape, device=w.device).index_add_(0, keys, dy).mul_(c["scale"])
        if s["padding"] is not None:
            dw[s["padding"]] = 0.0
        got["dweight"] = dw.to(w.dtype)
        if at is not None:
            dp = torch.zeros(s["position_weight"].shape, device=w.device).index_add_(0, at.reshape(-1), dy)
            got["dposition_weight"] = dp.to(w.dtype)
    return got


def _kept(rows, dim, p, seed):
    """[rows, dim]: 1 / (1 - p) where an element is kept, else 0 (32-bit words held in 64-bit numbers, whose products
    may pass the sign bit: the lower 64 bits are right all the same)."""
    word = 0xFFFFFFFF
    groups = -(-dim // 8)
    i = torch.arange(rows * groups, device=seed.device)
    c0, c1 = i & word, i >> 32
    c2, c3 = (seed[1] & word).expand_as(i), ((seed[1] >> 32) & word).expand_as(i)
    k0, k1 = seed[0] & word, (seed[0] >> 32) & word
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & word) ^ c1 ^ k0, b & word, ((a >> 32) & word) ^ c3 ^ k1, a & word
        k0, k1 = (k0 + 0x9E3779B9) & word, (k1 + 0xBB67AE85) & word
    numbers = torch.stack([half for c in (c0, c1, c2, c3) for half in (c & 0xFFFF, c >> 16)], 1)
    least = round(65536 * p)
    keep = numbers.view(rows, groups * 8)[:, :dim] >= least
    return keep.float() * (65536.0 / (65536 - least))


def _plain_dropout(s):
    c, x = s["case"], s["x"]
    k = _kept(c["rows"], c["dim"], c["p"], s["seed"])
    return {"y": (x.float() * k).to(x.dtype), "dx": (s["dy"].float() * k).to(x.dtype)}


def _plain_norm(s):
    c, r = s["case"], s["residual"]
    k = _kept(c["rows"], c["dim"], c["p"], s["seed"])
    h = (r.float() + s["x"].float() * k).to(r.dtype)
    hf, w = h.float(), s["weight"].float()
    mean = hf.mean(-1, keepdim=True)
    centred = hf - mean
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    n = centred * rstd
    dy = s["dy"].float()
    dn = dy * w
    dh = rstd * (dn - dn.mean(-1, keepdim=True) - n * (dn * n).mean(-1, keepdim=True)) + s["dh"].float()
    return {"y": (n * w + s["bias"].float()).to(r.dtype), "h": h, "dx": (dh * k).to(s["x"].dtype),
            "dresidual": dh.to(r.dtype), "dweight": (dy * n).sum(0).to(r.dtype), "dbias": dy.sum(0).to(r.dtype)}


def _softmax(logits, targets):
    """(softmax, log-probabilities of the targets, which targets count, their columns)."""
    counted = targets != IGNORED
    at = targets.masked_fill(~counted, 0)[:, None]
    x = logits.float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    logp = (x.gather(1, at) - top - torch.log(total))[:, 0] * counted
    return e.div_(total), logp, counted, at


def _times(p, at, factor):
    """factor (one-hot - softmax), in the softmax's memory."""
    p.scatter_add_(1, at, torch.full(at.shape, -1.0, device=p.device))
    return p.mul_(-factor[:, None])


def _plain_policy(s):
    c = s["case"]
    p, logp, counted, at = _softmax(s["logits"], s["actions"])
    share = counted.float() / counted.sum()
    a, ratio = s["advantages"], torch.exp(logp - s["old"])
    held = ratio.clamp(1.0 - c["low"], 1.0 + c["high"])
    row = -torch.minimum(ratio * a, held * a)
    slope = torch.where(ratio * a <= held * a, -ratio * a, torch.zeros_like(a))
    if c["kl"]:
        gap = s["ref"] - logp
        row = row + c["kl"] * (torch.exp(gap) - gap - 1.0)
        slope = slope + c["kl"] * (1.0 - torch.exp(gap))
    return {"loss": (row * share).sum(), "dlogits": _times(p, at, slope * share).to(s["logits"].dtype), "logp": logp}


def _plain_preference(s):
    c, t = s["case"], s["targets"]
    p, logp, counted, at = _softmax(s["logits"].view(-1, c["vocab"]), t.reshape(-1))
    total = logp.double().view(t.shape).sum(1)  # of a thousand tokens and more: a difference of two such sums matters
    over = total - s["ref"].double()
    m = (c["beta"] * (over[: c["pairs"]] - over[c["pairs"]:])).float()
    loss = (torch.relu(-m) + torch.log(1.0 + torch.exp(-m.abs()))).mean()
    slope = -c["beta"] / c["pairs"] / (1.0 + torch.exp(m))
    slope = torch.cat([slope, -slope])[:, None] * counted.view(t.shape).float()
    return {"loss": loss, "dlogits": _times(p, at, slope.view(-1)).to(s["logits"].dtype).view(s["logits"].shape),
            "logp": total.float()}


@torch.no_grad()
def _plain(state):
    return {"embedding": _plain_embedding, "dropout": _plain_dropout, "norm": _plain_norm, "policy": _plain_policy,
            "preference": _plain_preference}[state["case"]["op"]](state)


def run(state):
    if own:
        return {"embedding": _own_embedding, "dropout": _own_dropout, "norm": _own_norm, "policy": _own_policy,
                "preference": _own_preference}[state["case"]["op"]](state)
    return _plain(state)


# ---------------------------------------------------------------------------------------
# what a pass cannot do without

BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


def work(case):
    c, e = case, BYTES[case["dtype"]]
    if c["op"] == "embedding":
        n, d = c["batch"] * c["tokens"], c["dim"]
        places = min(n, c["positions"]) if c["given"] else min(c["tokens"], c["positions"])
        nbytes = 8 * n * (2 if c["given"] else 1) + e * d * (min(n, c["vocab"]) + places + n)  # rows in, y out
        flops = 2 * n * d
        if c["train"]:  # y's gradient in, the tables' out
            nbytes += e * d * (n + c["vocab"] + c["positions"])
            flops += 2 * n * d
        return {"bytes": nbytes, "flops": flops}
    if c["op"] == "dropout":
        return {"bytes": 4 * e * c["rows"] * c["dim"] + 16, "flops": 4 * c["rows"] * c["dim"]}
    if c["op"] == "norm":
        s, size, w = BYTES[c["stream"]], c["rows"] * c["dim"], c["dim"] * BYTES[c["stream"]]
        # x and residual in, y and h out; dy and dh in, dx and dresidual out (h comes out of the forward half)
        return {"bytes": size * (2 * e + 6 * s) + 5 * w + 16, "flops": 26 * size}
    rows = c["rows"] if c["op"] == "policy" else 2 * c["pairs"] * c["tokens"]
    size = rows * c["vocab"]
    small = rows * (8 + 4 * (4 if c["kl"] else 3)) if c["op"] == "policy" else 8 * rows + 16 * c["pairs"]
    return {"bytes": 2 * e * size + small, "flops": 6 * size}


# ---------------------------------------------------------------------------------------
# the same in 64 bits: the definitions, with gradients by differentiation


def _high(a, m):
    """The upper 32 bits of the products of 32-bit numbers, from their halves."""
    al, ah, ml, mh = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
    middle = ((al * ml) >> 16) + al * mh
    middle2 = (middle & 0xFFFF) + ah * ml
    return ah * mh + (middle >> 16) + (middle2 >> 16)


def _exact_mask(c, seed):
    """[rows, dim] float64 factors, of the generator's definition word by word."""
    key, offset = (int(x) % 2 ** 64 for x in seed.tolist())
    per = (c["dim"] + 7) // 8
    counter = torch.arange(c["rows"], device=seed.device)[:, None] * per + torch.arange(per, device=seed.device)
    x = [counter % 2 ** 32, counter // 2 ** 32, torch.full_like(counter, offset % 2 ** 32),
         torch.full_like(counter, offset // 2 ** 32)]
    k = [key % 2 ** 32, key // 2 ** 32]
    for turn in range(10):
        h0, l0 = _high(x[0], 0xD2511F53), (x[0] * 0xD2511F53) % 2 ** 32
        h1, l1 = _high(x[2], 0xCD9E8D57), (x[2] * 0xCD9E8D57) % 2 ** 32
        x = [h1 ^ x[1] ^ ((k[0] + turn * 0x9E3779B9) % 2 ** 32), l1, h0 ^ x[3] ^ ((k[1] + turn * 0xBB67AE85) % 2 ** 32), l0]
    least = round(65536 * c["p"])
    factor = torch.zeros(c["rows"], per, 8, dtype=torch.float64, device=seed.device)
    for j in range(8):
        factor[:, :, j] = ((x[j // 2] // 2 ** (16 * (j % 2))) % 65536 >= least) / (1.0 - least / 65536)
    return factor.reshape(c["rows"], -1)[:, : c["dim"]]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "embedding":
        w = s["weight"].detach().double().requires_grad_(True)
        leaves, names = [w], ["dweight"]
        y = F.embedding(s["ids"], w, padding_idx=s["padding"]) * c["scale"]
        if c["positions"]:
            leaves.append(s["position_weight"].detach().double().requires_grad_(True))
            names.append("dposition_weight")
            y = y + (F.embedding(s["positions"], leaves[1]) if c["given"] else leaves[1][: c["tokens"]])
        got = {"y": y.detach()}
        if c["train"]:
            got.update(zip(names, torch.autograd.grad(y, leaves, s["dy"].double())))
        return got
    if c["op"] == "dropout":
        f = _exact_mask(c, s["seed"])
        return {"y": s["x"].detach().double() * f, "dx": s["dy"].double() * f}
    if c["op"] == "norm":
        f = _exact_mask(c, s["seed"])
        # the stream as it is kept: the sum in 32 bits, rounded to the stream's type
        h = (s["residual"].detach().float() + s["x"].detach().float() * f.float()).to(s["residual"].dtype)
        leaves = [t.detach().double().requires_grad_(True) for t in (h, s["weight"], s["bias"])]
        y = F.layer_norm(leaves[0], (c["dim"],), leaves[1], leaves[2], EPS)
        dh, dw, db = torch.autograd.grad(y, leaves, s["dy"].double())
        dh = dh + s["dh"].double()
        return {"y": y.detach(), "h": h.double(), "dx": dh * f, "dresidual": dh, "dweight": dw, "dbias": db}
    x = s["logits"].double().requires_grad_(True)
    if c["op"] == "policy":
        nll = F.cross_entropy(x, s["actions"], ignore_index=IGNORED, reduction="none")
        counted, a = s["actions"] != IGNORED, s["advantages"].double()
        ratio = torch.exp(-nll - s["old"].double())
        row = -torch.minimum(ratio * a, ratio.clamp(1.0 - c["low"], 1.0 + c["high"]) * a)
        if c["kl"]:
            gap = s["ref"].double() + nll
            row = row + c["kl"] * (torch.expm1(gap) - gap)
        loss = row[counted].mean()
        return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss, x)[0], "logp": -nll.detach()}
    nll = F.cross_entropy(x.view(-1, c["vocab"]), s["targets"].view(-1), ignore_index=IGNORED, reduction="none")
    logp = -nll.view(s["targets"].shape).sum(1)
    over = logp - s["ref"].double()
    loss = -F.logsigmoid(c["beta"] * (over[: c["pairs"]] - over[c["pairs"]:])).mean()
    return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss, x)[0], "logp": logp.detach()}
