"""The two operators in front of the sampler, as cases that can be timed: what produces a decode step's logits, and what a
request asks of them before a token is drawn.

``op`` names the operator:

* ``adjust``  ``Engine.adjust_logits``: softcap, repetition / frequency / presence penalty over the streams' resident
              histories, logit biases and grammar masks, from logits as the model left them to the rows that are sampled;
* ``head``    ``Head.logits``: the LM head with 4-bit weights and a scale per group, hidden states to fp32 logits.

``own`` chooses between the plain form in elementary torch operations and the library's calls.
"""
import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _adjust(name=None, **kw):
    c = dict(op="adjust", rows=1, vocab=65536, pad=0, type="f32", out="f32", hist=256, penalty=1.1, freq=0.5, pres=0.25, bias=8, masks="mixed", softcap=0.0)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def _head(name=None, **kw):
    c = dict(op="head", rows=1, vocab=65536, hidden=2048, group=32, pad=0, type="bf16", scale="f16")
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the smallest call: one stream in a grammar, a short history - launch and latency
        _adjust("adjust_one_row", rows=1, vocab=65536, hist=64),
        # a small server's decode step, bf16 logits, requests with and without a grammar
        _adjust("adjust_slots", rows=8, vocab=65536, type="bf16", hist=256),
        # a vocabulary that is not a multiple of anything, rows off 16-byte boundaries, fp16 in and out
        _adjust("adjust_ragged", rows=24, vocab=100003, pad=1, type="f16", out="f16", hist=300, bias=300),
        # the benchmark's headline shape: large vocabulary, final-logit softcap in front of everything
        _adjust("adjust_softcap", rows=64, vocab=262144, hist=512, softcap=30.0),
        # penalties over whole histories of long conversations, no grammar
        _adjust("adjust_long_history", rows=16, vocab=131072, type="bf16", hist=16384, masks="none"),
        # a whole box's batch on one GPU: the largest
        _adjust("adjust_box", rows=512, vocab=262144, type="bf16", hist=1024),
        # one stream's token on a small model: the smallest head
        _head("head_one_small", rows=1, vocab=65536, hidden=1024),
        # a small server's decode step
        _head("head_slots", rows=8, vocab=65536, hidden=2048),
        # odd vocabulary, hidden size that is a multiple of 32 and nothing more, fp16
        _head("head_ragged", rows=5, vocab=100003, hidden=2016, type="f16", pad=8),
        # one stream's token on a large vocabulary, coarse groups: nothing but the weights' bytes
        _head("head_one_large", rows=1, vocab=262144, hidden=2560, group=128, scale="bf16"),
        # the headline batch: 64 rows of a large vocabulary, fine groups
        _head("head_batch", rows=64, vocab=262144, hidden=2560),
        # speculative verification, eight windows of seventeen rows
        _head("head_windows", rows=136, vocab=65536, hidden=2048, group=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    vocab = _log_int(rng, 4096, 262144)
    if rng.random() < 0.6:   # most vocabularies are padded to a round number, the rest are what the tokenizer gave
        vocab = vocab // 128 * 128
    if rng.random() < 0.5:
        t = rng.choice(["f32", "bf16", "f16"])
        c = _adjust(vocab=vocab, type=t, out=rng.choice(["f32", "f32", t]), hist=_log_int(rng, 1, 32768), penalty=rng.choice([1.0, 1.05, 1.1, 1.3]),
                    freq=rng.choice([0.0, 0.2, 0.5, -0.5]), pres=rng.choice([0.0, 0.25, 1.0]), bias=rng.choice([0, 0, 1, 8, 300]),
                    masks=rng.choice(["mixed", "mixed", "all", "none"]), softcap=rng.choice([0.0, 0.0, 30.0]), pad=rng.choice([0, 0, 1, 8, 64]))
        c["rows"] = max(1, min(_log_int(rng, 1, 512), (256 * 262144) // vocab, (1 << 20) // c["hist"]))
        return c
    group = rng.choice([32, 32, 64, 128])
    c = _head(vocab=vocab, group=group, hidden=_log_int(rng, 256, 4096) // group * group, type=rng.choice(["bf16", "bf16", "f16"]),
              scale=rng.choice(["f16", "bf16"]), pad=rng.choice([0, 0, 1, 8]))
    c["hidden"] = max(group, min(c["hidden"], 262144 * 2560 // vocab // group * group))
    c["rows"] = _log_int(rng, 1, 136)
    c["rows"] = max(1, min(c["rows"], 64 * 262144 * 2560 // (c["vocab"] * c["hidden"])))
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    return gen


def _masks(c, gen):
    """One mask per row that is in a grammar, packed 32 tokens to a word, and the mask of every row (-1: none).  What
    grammars leave: now a handful of tokens (structure), now nearly all (the inside of a string), now something between."""
    R, V = c["rows"], c["vocab"]
    words = (V + 31) // 32
    if c["masks"] == "none":
        return None, None
    rows = torch.arange(R, dtype=torch.int32)
    which = rows if c["masks"] == "all" else torch.where(rows % 4 == 3, torch.full_like(rows, -1), rows - rows // 4)
    n = int((which >= 0).sum())
    share = torch.tensor([0.0005, 0.97, 0.3], device="cuda")[torch.arange(n, device="cuda") % 3]
    packed = torch.zeros(n, words, dtype=torch.int32, device="cuda")
    for bit in range(32):
        packed |= (torch.rand(n, words, device="cuda", generator=gen) < share[:, None]).to(torch.int32) << bit
    return packed, which.numpy()


def _histories(c, gen, logits):
    """[rows][hist] token ids with Zipf frequencies; one in eight is a token that the model rates highly now."""
    R, V, n = c["rows"], c["vocab"], c["hist"]
    u = torch.rand(R, n, device="cuda", generator=gen, dtype=torch.float64)
    ids = (float(V) ** u - 1.0).long().clamp_(0, V - 1)   # density about 1 / id
    top = torch.topk(logits.float(), min(16, V), dim=1).indices
    hot = torch.gather(top, 1, torch.randint(top.shape[1], (R, n), device="cuda", generator=gen))
    return torch.where(torch.rand(R, n, device="cuda", generator=gen) < 0.125, hot, ids)


def _prepare_adjust(c, seed):
    gen, R, V = _generator(seed), c["rows"], c["vocab"]
    z = torch.randn(R, V + c["pad"], device="cuda", generator=gen).mul_(3.0)
    z.scatter_add_(1, torch.randint(V, (R, 16), device="cuda", generator=gen), 8.0 + 6.0 * torch.rand(R, 16, device="cuda", generator=gen))
    if c["softcap"]:
        z.mul_(4.0)
    s = {"case": c, "logits": z.to(TYPES[c["type"]])[:, :V], "out": torch.empty(R, V + c["pad"], dtype=TYPES[c["out"]], device="cuda")[:, :V]}
    s["masks"], s["mask_rows"] = _masks(c, gen)
    s["ids"] = _histories(c, gen, s["logits"])
    # every fourth request has its penalties off
    off = torch.arange(R, device="cuda") % 4 == 1
    value = lambda on, none: torch.where(off, torch.full((R,), none, device="cuda"), torch.full((R,), on, device="cuda"))  # noqa: E731
    s["penalty"], s["freq"], s["pres"] = value(c["penalty"], 1.0), value(c["freq"], 0.0), value(c["pres"], 0.0)
    n = min(c["bias"], V)
    s["bias_ids"] = torch.rand(R, V, device="cuda", generator=gen).topk(n, dim=1).indices if n else torch.zeros(R, 0, dtype=torch.long, device="cuda")
    s["bias"] = torch.rand(R, n, device="cuda", generator=gen) * 20.0 - 10.0
    return s


def _prepare_head(c, seed):
    gen, R, V, K = _generator(seed), c["rows"], c["vocab"], c["hidden"]
    weights = torch.randint(256, (V, K // 2), dtype=torch.uint8, device="cuda", generator=gen)   # two to a byte, low four bits first
    scales = (0.5 + torch.rand(V, K // c["group"], device="cuda", generator=gen)) * (0.65 / K ** 0.5)
    hidden = torch.randn(R, K + c["pad"], device="cuda", generator=gen)
    return {"case": c, "weights": weights, "scales": scales.to(TYPES[c["scale"]]), "hidden": hidden.to(TYPES[c["type"]])[:, :K],
            "logits": torch.empty(R, V + c["pad"], device="cuda")[:, :V]}


def _engine(c, s):
    """The engine, the open streams with their histories and settings, and the loaded head that a server keeps."""
    import ferro_b200 as fb
    R, V = c["rows"], c["vocab"]
    adjust = c["op"] == "adjust"
    pool = 1024 + (R * (max(256, 1 << (c["hist"] - 1).bit_length()) + max(256, 1 << (2 * c["bias"]).bit_length())) if adjust else 0)
    s["engine"] = eng = fb.Engine(device=0, max_rows=R, max_vocab=V, max_hist_ids=pool)
    eng.set_cuda_stream(torch.cuda.current_stream().cuda_stream)
    if not adjust:
        s["head"] = eng.load_head(s["weights"], s["scales"])
        return
    eng.set_softcap(c["softcap"])
    p = fb.make_params(R)
    p["repetition_penalty"] = s["penalty"].cpu().numpy()
    p["seed"] = 1 + np.arange(R)
    s["sids"] = eng.open_streams(p)
    ids, freq, pres = s["ids"].to(torch.int32).cpu().numpy(), s["freq"].tolist(), s["pres"].tolist()
    bias_ids, bias = s["bias_ids"].to(torch.int32).cpu().numpy(), s["bias"].cpu().numpy()
    for r, sid in enumerate(s["sids"]):
        eng.history_set(int(sid), ids[r])
        eng.set_penalties(int(sid), freq[r], pres[r])
        eng.set_bias(int(sid), bias_ids[r], bias[r])


def prepare(case, seed):
    c = dict(case)
    s = _prepare_adjust(c, seed) if c["op"] == "adjust" else _prepare_head(c, seed)
    if own:
        _engine(c, s)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _plain_adjust(s):
    c, x = s["case"], s["logits"].float()
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    count = torch.zeros_like(x).scatter_add_(1, s["ids"], torch.ones_like(s["ids"], dtype=torch.float32))
    seen = count > 0
    p = s["penalty"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / p, x * p), x)
    x = torch.where(seen, x - (s["freq"][:, None] * count + s["pres"][:, None]), x)
    if s["bias_ids"].shape[1]:
        x = x.scatter_add(1, s["bias_ids"], s["bias"])
    if s["masks"] is not None:
        which = torch.as_tensor(s["mask_rows"], device="cuda").long()
        v = torch.arange(x.shape[1], device="cuda")
        allowed = (s["masks"][which.clamp(min=0)][:, v // 32] >> (v % 32)) & 1
        x = torch.where((allowed == 1) | (which < 0)[:, None], x, float("-inf"))
    return x.to(TYPES[c["out"]])


def _plain_head(s):
    w = s["weights"]
    q = torch.stack([w & 15, w >> 4], dim=2).view(w.shape[0], -1).float() - 8.0
    q = q.view(w.shape[0], -1, s["case"]["group"]) * s["scales"].float()[:, :, None]
    return s["hidden"].float() @ q.view(w.shape[0], -1).T


def run(s):
    if s["case"]["op"] == "adjust":
        if own:
            return s["engine"].adjust_logits(s["sids"], s["logits"], s["out"], masks=s["masks"], mask_rows=s["mask_rows"])
        return _plain_adjust(s)
    if own:
        return s["head"].logits(s["hidden"], s["logits"])
    return _plain_head(s)


def work(case):
    c = case
    R, V = c["rows"], c["vocab"]
    if c["op"] == "adjust":
        # logits, window ids, biases and mask bits once, the result once; a comparison and a select per logit, a tanh counted as 20
        masked = {"none": 0, "mixed": R - R // 4, "all": R}[c["masks"]]
        bytes_ = R * V * (SIZE[c["type"]] + SIZE[c["out"]]) + 4 * R * c["hist"] + 8 * R * c["bias"] + 4 * masked * ((V + 31) // 32)
        return {"bytes": bytes_, "flops": R * V * (2 + (20 if c["softcap"] else 0))}
    K = c["hidden"]
    return {"bytes": V * K // 2 + 2 * V * (K // c["group"]) + SIZE[c["type"]] * R * K + 4 * R * V, "flops": 2 * R * V * K}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_adjust(s):
    c, R, V = s["case"], s["case"]["rows"], s["case"]["vocab"]
    out = torch.empty(R, V, dtype=torch.float64, device="cuda")
    for r in range(R):
        x = s["logits"][r].double()
        if c["softcap"]:
            x = c["softcap"] * torch.tanh(x / c["softcap"])
        ids, times = torch.unique(s["ids"][r], return_counts=True)
        p, f, q = float(s["penalty"][r]), float(s["freq"][r]), float(s["pres"][r])
        y = x[ids]
        x[ids] = torch.where(y > 0, y / p, y * p) - f * times.double() - q
        x[s["bias_ids"][r]] += s["bias"][r].double()
        if s["masks"] is not None and s["mask_rows"][r] >= 0:
            words = s["masks"][int(s["mask_rows"][r])]
            bits = torch.stack([(words >> b) & 1 for b in range(32)], dim=1).reshape(-1)[:V]
            x[bits == 0] = float("-inf")
        out[r] = x
    return out


def _exact_head(s):
    c, K = s["case"], s["case"]["hidden"]
    x = s["hidden"].double()
    parts = []
    for v in range(0, c["vocab"], 16384):
        w, g = s["weights"][v:v + 16384], s["scales"][v:v + 16384].double()
        full = torch.empty(w.shape[0], K, dtype=torch.float64, device="cuda")
        full[:, 0::2] = (w % 16).double() - 8
        full[:, 1::2] = (w // 16).double() - 8
        full *= torch.repeat_interleave(g, c["group"], dim=1)
        parts.append(torch.einsum("mk,vk->mv", x, full))
    return torch.cat(parts, dim=1)


def exact(case, seed):
    c = dict(case)
    if c["op"] == "adjust":
        return _exact_adjust(_prepare_adjust(c, seed))
    return _exact_head(_prepare_head(c, seed))
