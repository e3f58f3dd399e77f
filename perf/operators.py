"""Measured cases of the paged-cache operators: appending rotated keys and values to a cache in pages, attention of new
tokens over that cache, and attention over whole prompts packed without padding.  `run` computes them in elementary torch
operations, or with this package's kernels where `own` is set."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ---------------------------------------------------------------------------------------------------------
def _append(name, inp, dtype, seqs, q, past, heads, hd, rot, page, lens):
    return {"name": name, "op": "append", "in": inp, "dtype": dtype, "seqs": seqs, "q_min": q[0], "q_max": q[1], "past_min": past[0],
            "past_max": past[1], "nqh": heads[0], "nkv": heads[1], "hd": hd, "rot": rot, "page": page, "lens": lens}


def _paged(name, dtype, seqs, q, past, heads, hd, page, window, lens):
    return {"name": name, "op": "paged", "dtype": dtype, "seqs": seqs, "q_min": q[0], "q_max": q[1], "past_min": past[0],
            "past_max": past[1], "nqh": heads[0], "nkv": heads[1], "hd": hd, "page": page, "window": window, "lens": lens}


def _packed(name, dtype, seqs, q, heads, hd, window, lens):
    return {"name": name, "op": "packed", "dtype": dtype, "seqs": seqs, "q_min": q[0], "q_max": q[1], "past_min": 0, "past_max": 0,
            "nqh": heads[0], "nkv": heads[1], "hd": hd, "window": window, "lens": lens}


def listed():
    return [
        # one decode step of a small batch: the f32 projections of the quantized matvec into an f16 cache
        _append("append 8 new tokens", "f32", "f16", 8, (1, 1), (40, 2000), (32, 8), 128, 128, 16, 1),
        # a serving step that mixes single tokens with pieces of prompts; part of each head rotated, small pages
        _append("append mixed step", "bf16", "bf16", 24, (1, 513), (0, 4000), (12, 4), 96, 64, 24, 2),
        # prompts of a large model entering the cache at once
        _append("append prompts", "f32", "bf16", 6, (700, 4096), (0, 0), (64, 8), 128, 128, 64, 3),
        # decode of one sequence: latency
        _paged("decode 1 x 2k", "f16", 1, (1, 1), (2047, 2047), (32, 8), 128, 16, 0, 4),
        # decode of a busy server: ragged lengths, cache traffic
        _paged("decode 64 ragged", "bf16", 64, (1, 1), (90, 8191), (64, 8), 128, 32, 0, 5),
        # decode at the end of one very long context: few rows, a long axis
        _paged("decode 1 x 128k", "f16", 1, (1, 1), (131000, 131000), (32, 8), 128, 64, 0, 6),
        # the next piece of long prompts, fed in pieces
        _paged("chunk 512 on 16k", "f16", 2, (400, 512), (8000, 15872), (32, 8), 128, 64, 0, 7),
        # a mixed step of a model with local attention and an odd group of heads
        _paged("chunk ragged window", "bf16", 16, (1, 200), (0, 5000), (14, 2), 64, 48, 1024, 8),
        # one prompt of an 8B-class model
        _packed("prompt 2048", "f16", 1, (2048, 2048), (32, 8), 128, 0, 9),
        # long ragged prompts
        _packed("prompts ragged 8k", "bf16", 2, (5001, 8192), (32, 8), 128, 0, 10),
        # wide heads
        _packed("prompts head 256", "bf16", 3, (65, 1500), (8, 4), 256, 0, 11),
        # many short prompts, every query head with its own keys
        _packed("prompts short", "f16", 16, (3, 90), (16, 16), 64, 0, 12),
    ]


def _log(rng, lo, hi):
    return lo if lo >= hi else min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "paged", "paged", "packed"])
    nkv = rng.choice([1, 2, 4, 8])
    heads = (nkv * rng.choice([1, 2, 3, 4, 5, 7, 8]), nkv)
    hd = rng.choice([32, 64, 64, 96, 128, 128, 128, 256])
    dtype = rng.choice(["f16", "bf16"])
    page = rng.choice([8, 16, 24, 32, 64, 80, 128, 256])
    lens = rng.randrange(1 << 20)
    if op == "append":
        seqs, inp = _log(rng, 1, 64), rng.choice(["f32", "f16", "bf16"])
        most = 700_000_000 // ((heads[0] + 2 * nkv) * hd * (DTYPES[inp].itemsize + 2))  # tokens that cost as much as the largest listed case
        q_max = _log(rng, 1, min(16000, most) // seqs)
        case = _append("", inp, dtype, seqs, (_log(rng, 1, q_max), q_max), (0, _log(rng, 1, 20000)), heads, hd, rng.choice([hd, hd, hd // 2]), page, lens)
        del case["name"]
        return case
    window, most = rng.choice([0, 0, 0, _log(rng, 16, 4096)]), 150_000_000_000 // (heads[0] * hd)  # (row, key) pairs of a head, likewise
    if op == "paged":
        seqs = _log(rng, 1, 64)
        q_max = rng.choice([1, 1, _log(rng, 2, 1 + 1000 // seqs)])
        past = _log(rng, 64, min(100_000, 300_000 // seqs, most // (seqs * q_max)))
        case = _paged("", dtype, seqs, (_log(rng, 1, q_max), q_max), (_log(rng, 1 + past // 50, past), past), heads, hd, page, window, lens)
    else:
        seqs = _log(rng, 1, 32)
        q_max = _log(rng, 1, min(8192, int(math.sqrt(2 * most / seqs))))
        case = _packed("", dtype, seqs, (_log(rng, 1, q_max), q_max), heads, hd, window, lens)
    del case["name"]
    return case


def _lengths(case):
    """Per sequence: new tokens, and keys with the new ones included; the first sequence has the most, the last the fewest."""
    rng, n = random.Random(case["lens"]), case["seqs"]
    q = [_log(rng, case["q_min"], case["q_max"]) for _ in range(n)]
    past = [_log(rng, case["past_min"], case["past_max"]) for _ in range(n)]
    q[-1], past[-1] = case["q_min"], case["past_min"]
    q[0], past[0] = case["q_max"], case["past_max"]
    return q, [a + b for a, b in zip(q, past)]


# ---- inputs --------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    q, kv = _lengths(case)
    dtype, nqh, nkv, hd = DTYPES[case["dtype"]], case["nqh"], case["nkv"], case["hd"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, dtype: torch.randn(*shape, device="cuda", generator=g, dtype=dtype)  # noqa: E731
    total = sum(q)
    cu = [0]
    for n in q:
        cu.append(cu[-1] + n)
    s = {"case": case, "max_q": max(q), "max_kv": max(kv), "cu_q": torch.tensor(cu, dtype=torch.int32, device="cuda")}
    if case["op"] == "packed":
        # the projections of a layer side by side, as one product leaves them
        qkv = normal(total, (nqh + 2 * nkv) * hd, dtype=dtype)
        s["q"], s["k"], s["v"] = qkv[:, :nqh * hd], qkv[:, nqh * hd:(nqh + nkv) * hd], qkv[:, (nqh + nkv) * hd:]
        s["out"] = torch.empty(total, nqh * hd, dtype=dtype, device="cuda")
        return s
    # a pool that has served other sequences before, its pages handed out in no order
    page, need = case["page"], [-(-n // case["page"]) for n in kv]
    n_pages = sum(need) + 5
    order = random.Random(seed).sample(range(n_pages), sum(need))
    table, at = torch.zeros(len(kv), max(need), dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    s["table"] = table.cuda()
    s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["kpages"], s["vpages"] = normal(n_pages, page, nkv, hd, dtype=dtype), normal(n_pages, page, nkv, hd, dtype=dtype)
    if case["op"] == "append":
        s["qkv"] = normal(total, (nqh + 2 * nkv) * hd, dtype=DTYPES[case["in"]])
        s["q_out"] = torch.empty(total, nqh * hd, dtype=dtype, device="cuda")
        s["theta"] = 10000.0
    else:
        s["q"] = normal(total, nqh * hd, dtype=dtype)
        s["out"] = torch.empty(total, nqh * hd, dtype=dtype, device="cuda")
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------
def _rows(cu, total):
    """The sequence of every row of the batch, and its place there."""
    row = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu, row.to(cu.dtype), right=True) - 1
    return seq, row - cu.long()[seq]


def _rotate(x, cos, sin, rot):
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rot:]], dim=-1)


def _plain_append(s):
    case = s["case"]
    nqh, nkv, hd, rot, page = case["nqh"], case["nkv"], case["hd"], case["rot"], case["page"]
    qkv, cu = s["qkv"], s["cu_q"]
    total = qkv.shape[0]
    seq, i = _rows(cu, total)
    pos = s["kv_len"].long()[seq] - (cu[1:] - cu[:-1]).long()[seq] + i
    freq = torch.pow(torch.tensor(s["theta"], dtype=torch.float64, device="cuda"), -2.0 * torch.arange(rot // 2, dtype=torch.float64, device="cuda") / rot)
    angle = pos.double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = qkv.float().view(total, nqh + 2 * nkv, hd)
    q, k = _rotate(x[:, :nqh], cos, sin, rot), _rotate(x[:, nqh:nqh + nkv], cos, sin, rot)
    at = s["table"].long()[seq, pos // page]
    s["kpages"][at, pos % page] = k.to(s["kpages"].dtype)
    s["vpages"][at, pos % page] = x[:, nqh + nkv:].to(s["vpages"].dtype)
    return q.reshape(total, nqh * hd).to(s["q_out"].dtype), s["kpages"], s["vpages"]


def _plain_attention(q, k, v, q_len, kv_len, window, scale):
    """q (seqs, rows, nkv, group, hd), k and v (seqs, keys, nkv, hd), padded; row i of a sequence is position kv_len - q_len + i."""
    pos = (kv_len - q_len)[:, None] + torch.arange(q.shape[1], device=q.device)
    key = torch.arange(k.shape[1], device=q.device)
    seen = key[None, None] <= pos[:, :, None]
    if window:
        seen &= key[None, None] > pos[:, :, None] - window
    x = torch.einsum("sqkgd,stkd->skgqt", q * scale, k)
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    x.sub_(x.amax(dim=-1, keepdim=True)).exp_()
    total = x.sum(dim=-1)
    return torch.einsum("skgqt,stkd->sqkgd", x, v) / total.permute(0, 3, 1, 2)[..., None]


def _plain_attn(s):
    case, cu = s["case"], s["cu_q"]
    nqh, nkv, hd = case["nqh"], case["nkv"], case["hd"]
    total, q_len = s["q"].shape[0], (cu[1:] - cu[:-1]).long()
    place = (cu[:-1].long()[:, None] + torch.arange(s["max_q"], device="cuda")).clamp_(max=total - 1)
    q = s["q"][place].float().view(case["seqs"], s["max_q"], nkv, nqh // nkv, hd)
    if case["op"] == "paged":
        kv_len = s["kv_len"].long()
        k, v = (p[s["table"].long()].view(case["seqs"], -1, nkv, hd)[:, :s["max_kv"]].float() for p in (s["kpages"], s["vpages"]))
    else:
        kv_len = q_len
        k, v = (x[place].float().view(case["seqs"], s["max_q"], nkv, hd) for x in (s["k"], s["v"]))
    out = _plain_attention(q, k, v, q_len, kv_len, case["window"], hd ** -0.5)
    seq, i = _rows(cu, total)
    return out[seq, i].reshape(total, nqh * hd).to(s["out"].dtype)


def _own(s):
    from nates_recipe_rs_b200 import quant_ops as ops
    case = s["case"]
    if case["op"] == "append":
        ops.gpu_rope_kv_append_paged_into(s["qkv"], s["q_out"], s["kpages"], s["vpages"], s["table"], s["cu_q"], s["kv_len"], case["nqh"], s["theta"],
                                          rotary_dim=case["rot"])
        return s["q_out"], s["kpages"], s["vpages"]
    if case["op"] == "packed":
        ops.gpu_gqa_attn_packed_into(s["q"], s["k"], s["v"], s["cu_q"], s["out"], case["nqh"], case["nkv"], case["hd"], s["max_q"], case["hd"] ** -0.5,
                                     window=case["window"])
        return s["out"]
    if "scratch" not in s:  # a server keeps its workspace
        s["scratch"] = ops.gpu_gqa_attn_paged_scratch(s["q"], s["kpages"], s["kv_len"], case["nqh"], s["max_q"], s["max_kv"])
    ops.gpu_gqa_attn_paged_into(s["q"], s["kpages"], s["vpages"], s["table"], s["cu_q"], s["kv_len"], s["out"], case["nqh"], s["max_q"], s["max_kv"],
                                case["hd"] ** -0.5, window=case["window"], scratch=s["scratch"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["case"]["op"] == "append" else _plain_attn(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    q, kv = _lengths(case)
    nqh, nkv, hd = case["nqh"], case["nkv"], case["hd"]
    total = sum(q)
    if case["op"] == "append":
        size = DTYPES[case["in"]].itemsize
        return {"bytes": total * (nqh + 2 * nkv) * hd * (size + 2), "flops": 3 * total * (nqh + nkv) * case["rot"]}
    window = case["window"] or 1 << 40
    pairs = sum(sum(min(p + 1, window) for p in range(t - n, t)) for n, t in zip(q, kv))
    keys = sum(min(t, window + n - 1) for n, t in zip(q, kv))
    return {"bytes": 2 * hd * (2 * total * nqh + 2 * keys * nkv), "flops": 4 * hd * nqh * pairs}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    q_len, kv_len = _lengths(case)
    nqh, nkv, hd = case["nqh"], case["nkv"], case["hd"]
    if case["op"] == "append":
        half, page = case["rot"] // 2, case["page"]
        k_new, v_new = s["kpages"].double(), s["vpages"].double()
        x = s["qkv"].double().view(-1, nqh + 2 * nkv, hd)
        q_new, at = x[:, :nqh].clone(), 0
        for i, (n, t) in enumerate(zip(q_len, kv_len)):
            pos = torch.arange(t - n, t, device="cuda")
            turn = torch.polar(torch.ones(n, half, dtype=torch.float64, device="cuda"),
                               pos.double()[:, None] * torch.exp(torch.arange(half, device="cuda").double() * (-2 * math.log(s["theta"]) / case["rot"])))
            y = x[at:at + n].clone()
            z = torch.complex(y[:, :nqh + nkv, :half], y[:, :nqh + nkv, half:2 * half]) * turn[:, None]
            y[:, :nqh + nkv, :half], y[:, :nqh + nkv, half:2 * half] = z.real, z.imag
            q_new[at:at + n] = y[:, :nqh]
            where = s["table"][i].long()[pos // page]
            k_new[where, pos % page], v_new[where, pos % page] = y[:, nqh:nqh + nkv], y[:, nqh + nkv:]
            at += n
        return q_new.reshape(-1, nqh * hd), k_new, v_new
    out, at = torch.empty(sum(q_len), nqh, hd, dtype=torch.float64, device="cuda"), 0
    for i, (n, t) in enumerate(zip(q_len, kv_len)):
        q = s["q"][at:at + n].double().view(n, nqh, hd)
        if case["op"] == "paged":
            k, v = (p[s["table"][i].long()].view(-1, nkv, hd)[:t].double() for p in (s["kpages"], s["vpages"]))
        else:
            k, v = (x[at:at + n].double().view(n, nkv, hd) for x in (s["k"], s["v"]))
        ahead = torch.arange(t, device="cuda")[None] - torch.arange(t - n, t, device="cuda")[:, None]
        hidden = ahead > 0
        if case["window"]:
            hidden |= ahead <= -case["window"]
        for h in range(nqh):
            y = q[:, h] @ k[:, h * nkv // nqh].T / math.sqrt(hd)
            y[hidden] = float("-inf")
            out[at:at + n, h] = torch.softmax(y, dim=-1) @ v[:, h * nkv // nqh]
        at += n
    return out.view(-1, nqh * hd)
