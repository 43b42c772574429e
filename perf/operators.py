"""The operators of the 4-bit KV cache, as cases to measure: decode attention over the cache, packed prompts into it,
rotary positions with three axes, and eviction by accumulated attention weight.

Shapes are the model's: 24 query heads in 4 groups of 6, head dimension 256, 64 rotary dimensions.  A row of the cache
(one position, one kv head, K or V) holds 256 values as codes -7..7 with one scale per group of 32: the group's largest
magnitude over 7, rounded to four significant bits.
"""
import math
import random

import numpy as np
import torch

own = False

HQ, HKV, GRP, HD, HALF = 24, 4, 6, 256, 32
BASE, EPS = 1.0e7, float(np.float32(1e-6))
ROW = 136                                # bytes of one held row: 128 of codes and 8 scales
SMAX = 896.0                             # the largest scale


# ---- cases -------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one user's chat at 2048 cached tokens: the latency of a single step
        {"name": "decode 1 x 2048", "op": "decode", "seqs": 1, "shortest": 2048, "longest": 2048, "mix": 0,
         "tracked": False},
        # a serving batch of 64 users with contexts of 512 to 32768
        {"name": "decode 64 x 512-32768", "op": "decode", "seqs": 64, "shortest": 512, "longest": 32768, "mix": 2,
         "tracked": False},
        # eight long documents of 131072 tokens
        {"name": "decode 8 x 131072", "op": "decode", "seqs": 8, "shortest": 131072, "longest": 131072, "mix": 0,
         "tracked": False},
        # users on a cache budget: odd lengths, the attention weights accumulated for a later eviction
        {"name": "decode 12 x 900-7777 tracked", "op": "decode", "seqs": 12, "shortest": 900, "longest": 7777,
         "mix": 5, "tracked": True},
        # one short question
        {"name": "prompt 142", "op": "prompt", "seqs": 1, "shortest": 142, "longest": 142, "prior": 0, "mix": 0,
         "image": 0, "interleaved": False},
        # a packed batch of questions about images, of odd lengths
        {"name": "prompts 11 x 1-1500 images", "op": "prompt", "seqs": 11, "shortest": 1, "longest": 1500, "prior": 0,
         "mix": 3, "image": 16, "interleaved": True},
        # the last chunk of a document that is read in pieces
        {"name": "prompt 2000 after 5555", "op": "prompt", "seqs": 1, "shortest": 2000, "longest": 2000,
         "prior": 5555, "mix": 0, "image": 0, "interleaved": False},
        # a whole document of 8192 tokens
        {"name": "prompt 8192", "op": "prompt", "seqs": 1, "shortest": 8192, "longest": 8192, "prior": 0, "mix": 0,
         "image": 0, "interleaved": False},
        # the new tokens of a small batch
        {"name": "rotate 7 float32", "op": "rotate", "tokens": 7, "type": "float32", "first": 131000, "image": 0,
         "interleaved": False},
        # a long prompt with an image
        {"name": "rotate 32768 bfloat16", "op": "rotate", "tokens": 32768, "type": "bfloat16", "first": 0,
         "image": 64, "interleaved": True},
        # one user at the end of the budget: the oldest light entries go
        {"name": "evict 1 x 4352 to 4096", "op": "evict", "seqs": 1, "shortest": 4352, "longest": 4352, "keep": 4096,
         "recent": 256, "mix": 0},
        # a batch of long prompts, thinned for decoding
        {"name": "evict 13 x 9000-32768 to 2048", "op": "evict", "seqs": 13, "shortest": 9000, "longest": 32768,
         "keep": 2048, "recent": 128, "mix": 7},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "rotate", "evict"])
    mix = rng.randrange(1 << 20)
    if op == "decode":
        seqs = _spread(rng, 1, 64)
        longest = _spread(rng, 1, min(131072, (1 << 20) // seqs))
        return {"op": op, "seqs": seqs, "shortest": rng.randint(max(1, longest // 16), longest), "longest": longest,
                "mix": mix, "tracked": rng.random() < 0.4}
    if op == "prompt":
        seqs = _spread(rng, 1, 16)
        longest = _spread(rng, 1, 6000 // seqs)
        return {"op": op, "seqs": seqs, "shortest": rng.randint(1, longest), "longest": longest,
                "prior": rng.choice([0, 0, rng.randint(1, 1500 // seqs + 1)]), "mix": mix,
                "image": rng.choice([0, 0, 5, 8, 14]), "interleaved": rng.random() < 0.5}
    if op == "rotate":
        return {"op": op, "tokens": _spread(rng, 1, 32768), "type": rng.choice(["float32", "bfloat16"]),
                "first": _spread(rng, 1, 1 << 20), "image": rng.choice([0, 7, 24]), "interleaved": rng.random() < 0.5}
    seqs = _spread(rng, 1, 24)
    longest = _spread(rng, 64, 240000 // seqs)
    shortest = rng.randint(longest // 2, longest)
    keep = rng.randint(2, shortest)
    return {"op": op, "seqs": seqs, "shortest": shortest, "longest": longest, "keep": keep,
            "recent": rng.randint(0, keep // 2), "mix": mix}


def _lengths(case):
    r = random.Random(case["mix"])
    return [r.randint(case["shortest"], case["longest"]) for _ in range(case["seqs"])]


def work(case):
    if case["op"] == "decode":
        lens = _lengths(case)
        n, b = sum(lens), len(lens)
        held = (n + b) * HKV * 2 * ROW               # read, and the new rows written
        io = b * 4 * (HQ * 2 * HD + 2 * HKV * HD + HQ * HD + 2 * HKV * HD)
        return {"bytes": held + io + (8 * HKV * (n + b) if case["tracked"] else 0),
                "flops": 4 * HQ * HD * (n + b)}
    if case["op"] == "prompt":
        lens = _lengths(case)
        t, p = sum(lens), case["prior"] * len(lens)
        io = t * (2 * (HQ * 2 * HD + 2 * HKV * HD + HQ * HD) + 12 + 4 * 2 * HKV * HD)
        return {"bytes": (t + p) * HKV * 2 * ROW + io,
                "flops": 4 * HQ * HD * sum(n * case["prior"] + n * (n + 1) // 2 for n in lens)}
    if case["op"] == "rotate":
        size = 4 if case["type"] == "float32" else 2
        return {"bytes": case["tokens"] * (2 * size * (HQ + HKV) * HD + 12), "flops": 8 * case["tokens"] * 28 * HD}
    lens = _lengths(case)
    kept = HKV * len(lens) * case["keep"]
    # every weight read, every kept row read and written, its index and weight written, the rows read back as values
    return {"bytes": 4 * HKV * sum(lens) + kept * (4 * ROW + 8) + kept * 2 * HD * 4, "flops": 0}


# ---- inputs ------------------------------------------------------------------------------------------------------
def _starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)


def _positions(lens, first, image, dev):
    """[tokens][3] positions of packed sequences that begin at `first`: text, one image of image x image patches (its
    time stands still, its rows and columns count), then text again from the largest position on."""
    n = torch.tensor(lens, device=dev)
    at = torch.arange(int(n.sum()), device=dev) - torch.repeat_interleave(n.cumsum(0) - n, n)
    side = torch.where(n > 2 * image * image, image, 0)
    side, a = torch.repeat_interleave(side, n), torch.repeat_interleave(n // 4, n)
    inside, after = (at >= a) & (at < a + side * side), at >= a + side * side
    k = (at - a).clamp(min=0)
    row, col = k // side.clamp(min=1), k % side.clamp(min=1)
    text = torch.where(after, at - side * side + side, at)
    t = torch.where(inside, a, text)
    h, w = torch.where(inside, a + row, text), torch.where(inside, a + col, text)
    return (torch.stack([t, h, w], 1) + first).to(torch.int32).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev).to(dtype)

    def layer():
        return 1 + 0.1 * normal(HD), 1 + 0.1 * normal(HD)

    s = {"op": case["op"]}
    if case["op"] == "rotate":
        t, dtype = case["tokens"], getattr(torch, case["type"])
        s |= {"pos": _positions([t], case["first"], case["image"], dev), "interleaved": case["interleaved"],
              "q_gate": normal(t, HQ, 2 * HD, dtype=dtype), "k": normal(t, HKV, HD, dtype=dtype), "norms": layer()}
        if own:
            s["ctx"] = _context(s["norms"], case["interleaved"])
            s["q_out"], s["k_out"] = torch.empty_like(s["q_gate"][..., :HD]).contiguous(), torch.empty_like(s["k"])
        return s

    lens = _lengths(case)
    s["norms"] = layer()
    held = [case["prior"]] * len(lens) if case["op"] == "prompt" else lens
    caps = [n + 1 for n in lens] if case["op"] == "decode" else [n + p for n, p in zip(lens, held)] \
        if case["op"] == "prompt" else lens + [case["keep"]] * len(lens)
    tracked = case["op"] == "evict" or case.get("tracked", False)
    if own:
        s["ctx"] = _context(s["norms"], case.get("interleaved", False))
        s["ctx"].cache_create_q4(caps, track=tracked)
    # the rows that the cache holds already: K as normalised and rotated, V with its few large channels
    loud = 1 + 7 * (torch.rand(HD, generator=g, device=dev) < 0.03)
    rows = []
    for i, n in enumerate(held):
        k, v = normal(n, HKV, HD), normal(n, HKV, HD) * loud
        if own and n:
            s["ctx"].kv_import(0, i, k, v)
        if not own:
            rows.append([_pack(*_quantise(x.double())) for x in (k, v)])
    if not own:
        s["k_held"], s["v_held"] = ([torch.cat([r[j][m] for r in rows]) for m in (0, 1)] for j in (0, 1))
    start = _starts(held)
    s["lens"], s["start"] = torch.tensor(held, device=dev), torch.tensor(start[:-1], device=dev)
    s["longest"] = max(held)
    if tracked:
        # what decoding has left: a few entries draw most of the attention, some none
        n = int(start[-1]) * HKV
        s["weights"] = 1e-3 * torch.exp(2.5 * normal(n)) * (torch.rand(n, generator=g, device=dev) > 0.02)
    if case["op"] == "decode":
        b = len(lens)
        s |= {"q_gate": normal(b, HQ, 2 * HD), "k": normal(b, HKV, HD), "v": normal(b, HKV, HD) * loud,
              "pos": s["lens"][:, None].expand(b, 3).contiguous(), "tracked": tracked, "interleaved": False}
        if own:
            s |= {"host_lens": lens, "ids": list(range(b)), "out": torch.empty(b, HQ * HD, device=dev),
                  "rows": torch.empty(2, b, HKV, HD, device=dev)}
            if tracked:
                s["new_weights"] = torch.empty((int(start[-1]) + b) * HKV, device=dev)
    elif case["op"] == "prompt":
        t, bf = sum(lens), torch.bfloat16
        s |= {"q_gate": normal(t, HQ, 2 * HD, dtype=bf), "k": normal(t, HKV, HD, dtype=bf),
              "v": (normal(t, HKV, HD) * loud).to(bf), "new": torch.tensor(lens, device=dev),
              "pos": _positions(lens, case["prior"], case["image"], dev), "interleaved": case["interleaved"]}
        if own:
            s |= {"host_lens": held, "host_new": lens, "ids": list(range(len(lens))),
                  "out": torch.empty(t, HQ * HD, device=dev, dtype=bf), "rows": torch.empty(2, t, HKV, HD, device=dev)}
    else:
        s |= {"keep": case["keep"], "recent": case["recent"]}
        if own:
            b, keep = len(lens), case["keep"]
            s |= {"ids": list(range(b)), "into": list(range(b, 2 * b)),
                  "kept": torch.empty(b * HKV * keep, device=dev, dtype=torch.int32),
                  "rows": torch.empty(2, b * keep, HKV, HD, device=dev),
                  "new_weights": torch.empty(b * HKV * keep, device=dev)}
            s["ctx"].kv_set_weights_q4(0, s["ids"], s["weights"])
    return s


def _context(norms, interleaved):
    import daiza_b200 as dz
    ctx = dz.Context(torch.cuda.current_device(), dz.default_config(n_layers=1, full_attention_interval=1))
    ctx.set_attn_params(0, norms[0].cpu().numpy(), norms[1].cpu().numpy())
    ctx.set_rope_axes((11, 11, 10), interleaved)
    return ctx


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return {"decode": _own_decode, "prompt": _own_prompt, "rotate": _own_rotate, "evict": _own_evict}[s["op"]](s)
    return {"decode": _decode, "prompt": _prompt, "rotate": _rotate, "evict": _evict}[s["op"]](s)


def _own_decode(s):
    ctx, ids, lens = s["ctx"], s["ids"], s["host_lens"]
    for i, n in zip(ids, lens):              # each pass takes the same step again: back to the lengths before it
        ctx.kv_truncate(0, i, n)
    if s["tracked"]:
        ctx.kv_set_weights_q4(0, ids, s["weights"])
    ctx.gqa_decode_q4(0, ids, s["q_gate"], s["k"], s["v"], s["out"])
    ctx.kv_rows_q4(0, ids, lens, [1] * len(ids), s["rows"][0], s["rows"][1])
    got = {"out": s["out"], "k": s["rows"][0], "v": s["rows"][1]}
    if s["tracked"]:
        ctx.kv_weights_q4(0, ids, s["new_weights"])
        got["weights"] = s["new_weights"]
    return got


def _own_prompt(s):
    ctx, ids = s["ctx"], s["ids"]
    for i, n in zip(ids, s["host_lens"]):
        ctx.kv_truncate(0, i, n)
    ctx.gqa_prefill_q4(0, ids, s["host_new"], s["q_gate"], s["k"], s["v"], s["out"], pos=s["pos"])
    ctx.kv_rows_q4(0, ids, s["host_lens"], s["host_new"], s["rows"][0], s["rows"][1])
    return {"out": s["out"], "k": s["rows"][0], "v": s["rows"][1]}


def _own_rotate(s):
    s["ctx"].qk_mrope(0, s["pos"], s["q_gate"], s["k"], s["q_out"], s["k_out"])
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_evict(s):
    ctx, n = s["ctx"], len(s["ids"])
    ctx.kv_evict_q4(0, s["ids"], [s["keep"]] * n, [s["recent"]] * n, kept=s["kept"], into=s["into"])
    ctx.kv_rows_q4(0, s["into"], [0] * n, [s["keep"]] * n, s["rows"][0], s["rows"][1])
    ctx.kv_weights_q4(0, s["into"], s["new_weights"])
    return {"kept": s["kept"], "k": s["rows"][0], "v": s["rows"][1], "weights": s["new_weights"]}


# ---- the plain form ----------------------------------------------------------------------------------------------
def _quantise(x):
    """Codes -7..7 and scales of rows x [..., 256] in 64 bits: values next to a border fall the same way everywhere."""
    x = torch.where(torch.isnan(x), 0.0, x).unflatten(-1, (HD // 32, 32))
    t = (x.abs().amax(-1) / 7).clamp(max=SMAX)
    step = torch.exp2((torch.frexp(t)[1].clamp(min=-13) - 4).double())
    scale = torch.round(t / step) * step
    scale = scale.clamp(max=SMAX)
    code = torch.round(x / torch.where(scale > 0, scale, 1.0)[..., None]).clamp(-7, 7)
    return torch.where(scale[..., None] > 0, code, 0.0).flatten(-2), scale


def _pack(code, scale):
    n = (code + 8).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), scale.to(torch.float16)


def _values(held):
    code = torch.stack([held[0] & 15, held[0] >> 4], -1).flatten(-2).to(torch.float32) - 8
    return (code.unflatten(-1, (HD // 32, 32)) * held[1].to(torch.float32)[..., None]).flatten(-2)


def _axis(interleaved, dev):
    pair = torch.arange(HALF, device=dev)
    if interleaved:                          # t h w t h w ..., time where an axis has used up its pairs
        return torch.where((pair % 3 == 1) & (pair < 33), 1, torch.where((pair % 3 == 2) & (pair < 30), 2, 0))
    return (pair >= 11).long() + (pair >= 22).long()


def _turned(x, norm, pos, interleaved):
    """RMS-normalised and rotated rows x [tokens][heads][256], in x's own precision; the angles always in 64 bits."""
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * norm.to(x.dtype)
    pair = torch.arange(HALF, device=x.device, dtype=torch.float64)
    angle = pos[:, _axis(interleaved, x.device)].double() * BASE ** (-2 * pair / 64)
    c, sn = torch.cos(angle).to(x.dtype)[:, None], torch.sin(angle).to(x.dtype)[:, None]
    a, b, rest = x[..., :HALF], x[..., HALF:2 * HALF], x[..., 2 * HALF:]
    return torch.cat([a * c + b * sn, b * c + a * sn, rest], -1)


def _new_rows(s):
    k = _quantise(_turned(s["k"].double(), s["norms"][1], s["pos"], s["interleaved"]))
    return _values(_pack(*k)), _values(_pack(*_quantise(s["v"].double())))


def _decode(s):
    b, n = len(s["lens"]), s["longest"]
    q = _turned(s["q_gate"][..., :HD], s["norms"][0], s["pos"], s["interleaved"]) / 16
    q = q.reshape(b, HKV, GRP, HD)
    k, v = _new_rows(s)
    j = torch.arange(n, device=q.device)
    there = j < s["lens"][:, None]
    at = torch.where(there, s["start"][:, None] + j, 0)
    keys = _values(s["k_held"])[at].permute(0, 2, 3, 1)
    score = torch.where(there[:, None, None], q @ keys, -math.inf)
    del keys
    score = torch.cat([score, (q * k[:, :, None]).sum(-1, keepdim=True)], -1)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = p[..., :n] @ _values(s["v_held"])[at].permute(0, 2, 1, 3) + p[..., n:] * v[:, :, None]
    out = o.reshape(b, HQ, HD) / (1 + torch.exp(-s["q_gate"][..., HD:]))
    got = {"out": out.reshape(b, HQ * HD), "k": k, "v": v}
    if s["tracked"]:
        new = p.sum(2)                                              # [b][kv head][position]
        w, lens = s["weights"], s["lens"]
        of = torch.repeat_interleave(torch.arange(b, device=q.device), HKV * (lens + 1))
        i = torch.arange(len(of), device=q.device) - HKV * (s["start"] + torch.arange(b, device=q.device))[of]
        h, j = i // (lens[of] + 1), i % (lens[of] + 1)
        old = w[torch.where(j < lens[of], HKV * s["start"][of] + h * lens[of] + j, 0)]
        got["weights"] = new[of, h, torch.where(j < lens[of], j, n)] + torch.where(j < lens[of], old, 0.0)
    return got


def _prompt(s):
    t, new, lens = len(s["pos"]), s["new"], s["lens"]
    dev = new.device
    q = _turned(s["q_gate"][..., :HD].float(), s["norms"][0], s["pos"], s["interleaved"]) / 16
    k, v = _new_rows(s)
    seq = torch.arange(len(new), device=dev)
    of_new, of_old = torch.repeat_interleave(seq, new), torch.repeat_interleave(seq, lens)
    at_new = torch.arange(t, device=dev) - (new.cumsum(0) - new)[of_new] + lens[of_new]
    at_old = torch.arange(len(of_old), device=dev) - s["start"][of_old]
    keys, values = torch.cat([_values(s["k_held"]), k]), torch.cat([_values(s["v_held"]), v])
    of, at = torch.cat([of_old, of_new]), torch.cat([at_old, at_new])
    sees = (of_new[:, None] == of) & (at <= at_new[:, None])
    q = q.reshape(t, HKV, GRP, HD).permute(1, 2, 0, 3).reshape(HKV, GRP * t, HD)
    score = (q @ keys.permute(1, 2, 0)).reshape(HKV, GRP, t, len(at)).masked_fill_(~sees, -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = p.reshape(HKV, GRP * t, len(at)) @ values.permute(1, 0, 2)
    o = (o.reshape(HKV, GRP, t, HD) / p.sum(-1, keepdim=True)).permute(2, 0, 1, 3).reshape(t, HQ, HD)
    out = o / (1 + torch.exp(-s["q_gate"][..., HD:].float()))
    return {"out": out.reshape(t, HQ * HD).to(s["q_gate"].dtype), "k": k, "v": v}


def _rotate(s):
    dtype = s["k"].dtype
    q = _turned(s["q_gate"][..., :HD].float(), s["norms"][0], s["pos"], s["interleaved"]) / 16
    return {"q": q.to(dtype), "k": _turned(s["k"].float(), s["norms"][1], s["pos"], s["interleaved"]).to(dtype)}


def _evict(s):
    lens, n, keep = s["lens"], s["longest"], s["keep"]
    b, dev = len(lens), lens.device
    j, h = torch.arange(n, device=dev), torch.arange(HKV, device=dev)
    at = HKV * s["start"][:, None, None] + h[:, None] * lens[:, None, None] + j
    there = (j < lens[:, None])[:, None].expand(b, HKV, n)
    w = s["weights"][torch.where(there, at, 0)]
    rank = torch.where(j >= (lens - s["recent"])[:, None, None], math.inf, w)
    order = torch.sort(torch.where(there, rank, -1.0), dim=-1, descending=True, stable=True)[1][..., :keep]
    kept = torch.sort(order, dim=-1)[0]                             # [b][kv head][keep], ascending
    row = (s["start"][:, None, None] + kept).transpose(1, 2)        # [b][keep][kv head]
    k, v = (_values((x[0][row, h], x[1][row, h])).reshape(b * keep, HKV, HD) for x in (s["k_held"], s["v_held"]))
    return {"kept": kept.reshape(-1).to(torch.int32), "k": k, "v": v, "weights": torch.gather(w, 2, kept).reshape(-1)}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    """By the definition, a sequence and a head at a time, in numpy's and torch's 64 bits."""
    s = prepare(case, seed)
    dev = s["norms"][0].device
    f = torch.float64

    def held(x):                             # code * scale, from the bytes
        lo, hi = (x[0] & 15).to(f) - 8, (x[0] >> 4).to(f) - 8
        return torch.stack([lo, hi], -1).reshape(*x[0].shape[:-1], HD) * x[1].to(f).repeat_interleave(32, -1)

    def hold(x):                             # the nearest held row of each row
        group = x.reshape(-1, 32)
        t = np.minimum(group.abs().amax(1).cpu().numpy() / 7, SMAX)
        m, e = np.frexp(t)
        ulp = np.ldexp(1.0, np.maximum(e, -13) - 4)
        sc = torch.tensor(np.rint(t / ulp) * ulp, device=dev)[:, None]
        return torch.where(sc > 0, torch.clamp(torch.round(group / sc), -7, 7) * sc, 0.0).reshape(x.shape)

    def turn(x, norm, pos):
        x = x.to(f)
        x = x * (x.pow(2).sum(-1, keepdim=True) / HD + EPS).pow(-0.5) * norm.to(f)
        y = x.clone()
        for i in range(HALF):
            if case.get("interleaved", False):
                ax = 1 if i % 3 == 1 and i < 33 else 2 if i % 3 == 2 and i < 30 else 0
            else:
                ax = 0 if i < 11 else 1 if i < 22 else 2
            th = pos[:, ax].to(f) / 10.0 ** (7 * i / 32)
            c, sn = th.cos()[:, None], th.sin()[:, None]
            y[..., i] = x[..., i] * c + x[..., i + HALF] * sn
            y[..., i + HALF] = x[..., i + HALF] * c + x[..., i] * sn
        return y

    if case["op"] == "rotate":
        return {"q": turn(s["q_gate"][..., :HD], s["norms"][0], s["pos"]) / 16, "k": turn(s["k"], s["norms"][1], s["pos"])}
    lens = s["lens"].tolist()
    start = s["start"].tolist()
    if case["op"] == "evict":
        kept, k, v, weights = [], [], [], []
        w = s["weights"].cpu().numpy()
        for n, a in zip(lens, start):
            mine = w[HKV * a:HKV * (a + n)].reshape(HKV, n)
            old = n - case["recent"]
            for h in range(HKV):
                best = np.lexsort((np.arange(old), -mine[h, :old]))[:case["keep"] - case["recent"]]
                kept.append(np.concatenate([np.sort(best), np.arange(old, n)]).astype(np.int32))
                weights.append(mine[h][kept[-1]].astype(np.float64))
            row = torch.tensor(a + np.stack(kept[-HKV:]), device=dev)
            for to, x in ((k, s["k_held"]), (v, s["v_held"])):
                to.append(torch.stack([held((x[0][row[h], h], x[1][row[h], h])) for h in range(HKV)], 1))
        return {"kept": np.concatenate(kept), "k": torch.cat(k), "v": torch.cat(v), "weights": np.concatenate(weights)}
    q = turn(s["q_gate"][..., :HD], s["norms"][0], s["pos"]) / 16
    gate = torch.sigmoid(s["q_gate"][..., HD:].to(f))
    k_new, v_new = hold(turn(s["k"], s["norms"][1], s["pos"])), hold(s["v"].to(f))
    new = [1] * len(lens) if case["op"] == "decode" else _lengths(case)
    out, weights, t0 = torch.empty(len(q), HQ, HD, dtype=f, device=dev), [], 0
    for n, a, t in zip(lens, start, new):
        k_old, v_old = (held((x[0][a:a + n], x[1][a:a + n])) for x in (s["k_held"], s["v_held"]))
        later = torch.ones(t, n + t, dtype=torch.bool, device=dev).triu(n + 1)
        for h in range(HKV):
            keys = torch.cat([k_old[:, h], k_new[t0:t0 + t, h]])
            values = torch.cat([v_old[:, h], v_new[t0:t0 + t, h]])
            total = torch.zeros(n + t, dtype=f, device=dev)
            for i in range(GRP * h, GRP * h + GRP):
                p = torch.softmax((q[t0:t0 + t, i] @ keys.T).masked_fill(later, -math.inf), -1)
                out[t0:t0 + t, i] = p @ values * gate[t0:t0 + t, i]
                total += p[0] if case["op"] == "decode" else 0
            if case.get("tracked", False):
                total[:n] += s["weights"][HKV * a + h * n:HKV * a + h * n + n]
                weights.append(total)
        t0 += t
    got = {"out": out.reshape(len(q), HQ * HD), "k": k_new, "v": v_new}
    return got | {"weights": torch.cat(weights)} if weights else got
