"""Measured cases of the paged int8 key/value cache: ``paged_append`` and ``paged_attention``.

A batch is ragged: sequence b brings ``query_starts[b + 1] - query_starts[b]`` new tokens and holds
``kv_lens[b]`` keys once they are appended.  Position p of sequence b lies in page
``block_table[b, p // page]``, row ``p % page``, of pools laid out [pages, kv_heads, page, dim].

The plain forms are elementary torch operations in 32 bits, rounded once at the end; with ``own`` the same
state goes through the framework's entry points.  An int8 pool is returned as it is (its whole numbers are
what the integer products consume, and the arithmetic up to the rounding is fixed operation by operation, so
both sides have to agree exactly); an int8 context is returned as the values of its units, and has no value
in 64 bits: its last step is a rounding to whole units, where a tie moves a whole unit.
"""
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"int8": torch.int8, "fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_SIZES = {"int8": 1, "fp16": 2, "bf16": 2, "fp32": 4}


def _append(name, batch, new, context, heads, kv_heads, dim, page, dtype, rotary, rotary_dim, layout):
    return {"name": name, "op": "append", "batch": batch, "new": new, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "rotary": rotary,
            "rotary_dim": rotary_dim, "layout": layout}


def _attention(name, batch, new, context, heads, kv_heads, dim, page, out, layout):
    return {"name": name, "op": "attention", "batch": batch, "new": new, "context": context, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "out": out, "layout": layout}


def listed():
    return [
        # One decode step of OPT-30B at batch 8: the int8 keys and values of the fused projection, as they are.
        _append("append_decode_opt30b", 8, 1, 640, 0, 56, 128, 16, "int8", "none", 0, "even:1"),
        # The 512-token prompts of the same model.
        _append("append_prompts_opt30b", 8, 512, 0, 0, 56, 128, 16, "int8", "none", 0, "even:2"),
        # A few drafted tokens per sequence of a model with rotary positions and shared key heads.
        _append("append_rotated_drafts", 16, 5, 1500, 32, 8, 128, 16, "bf16", "half", 128, "ragged:3"),
        # Long prompt chunks behind linears with fp32 output, part of each head rotated in neighbouring pairs.
        _append("append_rotated_chunks", 4, 2048, 6000, 40, 40, 128, 64, "fp32", "pairs", 64, "ragged:4"),
        # One sequence, one token, a short context (OPT-1.3B heads): latency.
        _attention("decode_single_opt1b3", 1, 1, 500, 32, 32, 64, 16, "int8", "even:5"),
        # A decode step of OPT-30B at batch 8 between its prompts' end and 128 tokens later.
        _attention("decode_opt30b", 8, 1, 640, 56, 56, 128, 16, "int8", "near:6"),
        # A full decode batch of unequal contexts, four query heads per key head.
        _attention("decode_ragged_batch", 64, 1, 8192, 32, 8, 128, 64, "bf16", "ragged:7"),
        # Two very long contexts, eight query heads per key head: the work is along the keys.
        _attention("decode_long", 2, 1, 131072, 64, 8, 128, 128, "fp16", "near:8"),
        # Drafted tokens are verified: up to five new tokens per sequence (OPT-2.7B heads, 80 wide).
        _attention("verify_drafts_opt2b7", 16, 5, 1999, 32, 32, 80, 32, "fp16", "ragged:9"),
        # The 512-token prompts of OPT-30B.
        _attention("prompts_opt30b", 8, 512, 0, 56, 56, 128, 16, "int8", "even:10"),
        # A chunk of a long prompt behind what is cached of it.
        _attention("chunk_long_prompt", 1, 2048, 14336, 32, 8, 128, 64, "bf16", "even:11"),
        # A batch that mixes one prompt chunk with decoding sequences (OPT-1.3B heads).
        _attention("mixed_batch_opt1b3", 16, 777, 3300, 32, 32, 64, 16, "bf16", "mixed:12"),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], even in its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    seed = rng.randrange(1 << 20)
    dim = rng.choice((64, 80, 128, 128))
    page = rng.choice((16, 32, 64, 128))
    kv_heads = rng.choice((1, 2, 4, 8, 12, 20, 32, 40))
    group = rng.choice((1, 1, 2, 4, 5, 8)) if kv_heads <= 8 else 1
    heads = kv_heads * group
    kind = rng.choice(("append", "decode", "decode", "chunk", "chunk", "mixed"))
    if kind == "append":
        dtype = rng.choice(("int8", "fp16", "bf16", "fp32"))
        rotary = rng.choice(("none", "half", "pairs"))
        rotary_dim = 0 if rotary == "none" else rng.choice((dim, dim // 2 // 16 * 16))
        new = _between(rng, 1, 2048)
        batch = _between(rng, 1, max(1, min(64, (500 << 20) // (new * (heads + 2 * kv_heads) * dim * _SIZES[dtype]))))
        return {k: v for k, v in _append("", batch, new, _between(rng, 1, 4000), heads if rng.random() < 0.7 else 0,
                                         kv_heads, dim, page, dtype, rotary, rotary_dim,
                                         rng.choice(("even:%d", "ragged:%d")) % seed).items() if k != "name"}
    if kind == "decode":
        context = _between(rng, 1, 65536)
        new = rng.choice((1, 1, 1, 2, 4, 7))
        batch = _between(rng, 1, max(1, min(96, (500 << 20) // (2 * context * kv_heads * dim))))
        layout = rng.choice(("even:%d", "near:%d", "ragged:%d")) % seed
        out = rng.choice(("int8", "fp16", "bf16"))
    elif kind == "chunk":
        new, context = _between(rng, 8, 2048), _between(rng, 1, 12000)
        batch = _between(rng, 1, max(1, min(8, (1 << 29) // (new * (new + context) * heads))))
        layout = rng.choice(("even:%d", "ragged:%d")) % seed
        out = rng.choice(("int8", "fp16", "bf16"))
    else:
        new, context = _between(rng, 16, 1024), _between(rng, 16, 4000)
        batch = _between(rng, 2, max(2, min(24, (1 << 30) // (new * (new + context) * heads))))
        layout = "mixed:%d" % seed
        out = rng.choice(("fp16", "bf16"))
    return {k: v for k, v in _attention("", batch, new, context, heads, kv_heads, dim, page, out, layout).items()
            if k != "name"}


def _lengths(case):
    """(new tokens, keys) of each sequence: a property of the case, not of the seed."""
    kind, seed = case["layout"].split(":")
    r = random.Random(int(seed))
    batch, new, context = case["batch"], case["new"], case["context"]
    if kind == "even":
        lens = [(new, context + new)] * batch
    elif kind == "near":  # contexts within a fifth of the longest
        lens = [(new, new + r.randint(context - context // 5, context)) for _ in range(batch)]
    elif kind == "ragged":
        lens = [(t, t + r.randint(0, context)) for t in (r.randint(1, new) for _ in range(batch))]
        lens[0] = (new, new + context)
    else:  # one chunk among single tokens
        lens = [(1, 1 + r.randint(0, context)) for _ in range(batch)]
        lens[r.randrange(batch)] = (new, new + context)
    return [t for t, _ in lens], [n for _, n in lens]


def _f32(x):
    return torch.tensor(x, dtype=torch.float32).item()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, keys = _lengths(case)
    batch, tokens, page, dim = case["batch"], sum(new), case["page"], case["dim"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    table_width = max(-(-n // page) for n in keys)
    pages = sum(-(-n // page) for n in keys) + 3

    def activations(n, h, dtype):
        x = torch.randn((n, h, dim), generator=g, device="cuda") * 40
        return x.round_().clamp_(-127, 127).to(torch.int8) if dtype == "int8" else (x * 0.03).to(_DTYPES[dtype])

    def pool():
        x = torch.empty((pages, kv_heads, page, dim), dtype=torch.int8, device="cuda")
        for i in range(0, pages, 4096):
            x[i:i + 4096] = (torch.randn(x[i:i + 4096].shape, generator=g, device="cuda") * 40).round_().clamp_(-127, 127)
        return x

    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = torch.zeros((batch, table_width), dtype=torch.int32)
    for b, n in enumerate(keys):
        used = -(-n // page)
        table[b, :used] = torch.tensor(order[:used], dtype=torch.int32)
        del order[:used]
    starts = [0]
    for t in new:
        starts.append(starts[-1] + t)
    s = {"op": case["op"], "block_table": table.cuda(), "page": page, "dim": dim,
         "query_starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
         "kv_lens": torch.tensor(keys, dtype=torch.int32, device="cuda"),
         "max_query_len": max(new), "max_kv_len": max(keys), "k_pages": pool(), "v_pages": pool()}
    if case["op"] == "append":
        # the projections' output: q, k and v of a token side by side in one row
        qkv = activations(tokens, heads + 2 * kv_heads, case["dtype"])
        s["q"] = qkv[:, :heads] if heads else None
        s["k"], s["v"] = qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        s["alpha"] = {"q": 1.0, "k": 1.0, "v": 1.0} if case["dtype"] == "int8" and case["rotary"] == "none" else \
            {n: _f32((0.8 if case["dtype"] == "int8" else 33.0) * (1 + 0.1 * i)) for i, n in enumerate("qkv")}
        s["rotary"], s["interleaved"] = None, case["rotary"] == "pairs"
        if case["rotary"] != "none":
            rd = case["rotary_dim"]
            angle = torch.arange(max(keys), dtype=torch.float64, device="cuda")[:, None] * \
                10000.0 ** (-torch.arange(0, rd, 2, dtype=torch.float64, device="cuda") / rd)
            s["rotary"] = torch.cat((angle.cos(), angle.sin()), dim=1).float().contiguous()
    else:
        s["q"] = activations(tokens, heads, "int8")
        s["alpha_qk"] = _f32(2.0 / (1600.0 * dim ** 0.5))
        out = case["out"]
        # about the standard deviation of a context, in units of a calibrated int8 scale
        s["alpha_pv"] = _f32(0.02 if out != "int8" else 1.0 if max(keys) < 200 else 2.5)
        s["out_dtype"] = _DTYPES[out]
    return s


# ------------------------------------------------------------------------------------------- plain forms
def _places(s, tokens):
    """(sequence, position) of every new token."""
    i = torch.arange(tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["query_starts"][1:], i, right=True)
    return seq, s["kv_lens"][seq] - (s["query_starts"][seq + 1] - i)


def _rotate(x, table, interleaved):
    rd = table.shape[-1]
    c, sn = table[:, None, :rd // 2], table[:, None, rd // 2:]
    a, rest = x[..., :rd], x[..., rd:]
    x1, x2 = (a[..., 0::2], a[..., 1::2]) if interleaved else (a[..., :rd // 2], a[..., rd // 2:])
    y1, y2 = x1 * c - x2 * sn, x2 * c + x1 * sn
    y = torch.stack((y1, y2), dim=-1).flatten(-2) if interleaved else torch.cat((y1, y2), dim=-1)
    return torch.cat((y, rest), dim=-1)


def _whole(x):
    return x.round().clamp(-128, 127).to(torch.int8)


def _append_plain(s):
    seq, pos = _places(s, s["k"].shape[0])
    page = s["block_table"][seq, pos // s["page"]].long()
    row = (pos % s["page"]).long()
    q, k, v = None if s["q"] is None else s["q"].float(), s["k"].float(), s["v"].float()
    if s["rotary"] is not None:
        table = s["rotary"][pos]
        k = _rotate(k, table, s["interleaved"])
        q = None if q is None else _rotate(q, table, s["interleaved"])
    s["k_pages"][page, :, row] = _whole(k * s["alpha"]["k"])
    s["v_pages"][page, :, row] = _whole(v * s["alpha"]["v"])
    return {"q": None if q is None else _whole(q * s["alpha"]["q"]), "k": s["k_pages"], "v": s["v_pages"]}


def _attention_plain(s):
    n, heads, dim = s["q"].shape
    kv_heads = s["k_pages"].shape[1]
    group = heads // kv_heads
    batch, t_max = s["kv_lens"].shape[0], s["max_query_len"]
    starts, lens = s["query_starts"], s["kv_lens"]
    # padded queries [B, Hkv, G * T, D] and gathered keys [B, Hkv, S, D]
    t = torch.arange(t_max, device="cuda", dtype=torch.int32)
    q = s["q"][(starts[:-1, None] + t).clamp(max=n - 1)].float()
    q = q.view(batch, t_max, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * t_max, dim)
    table = s["block_table"].long()
    k = s["k_pages"][table].transpose(1, 2).reshape(batch, kv_heads, -1, dim).float()
    v = s["v_pages"][table].transpose(1, 2).reshape(batch, kv_heads, -1, dim).float()
    pos = lens[:, None] - (starts[1:] - starts[:-1])[:, None] + t  # [B, T]
    hidden = torch.arange(k.shape[2], device="cuda", dtype=torch.int32) > pos[..., None]
    scores = (q @ k.transpose(2, 3)).view(batch, kv_heads, group, t_max, -1)
    scores = (scores * s["alpha_qk"]).masked_fill_(hidden[:, None, None], float("-inf"))
    p = (scores - scores.amax(dim=-1, keepdim=True)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    ctx = p.view(batch, kv_heads, group * t_max, -1) @ v
    ctx = ctx.view(batch, kv_heads, group, t_max, dim) / total * s["alpha_pv"]
    seq, at = _places(s, n)
    row = at - pos[seq, 0]
    ctx = ctx.permute(0, 3, 1, 2, 4).reshape(batch, t_max, heads, dim)[seq, row]
    if s["out_dtype"] == torch.int8:
        return ctx.round().clamp(-128, 127).to(torch.float16)
    return ctx.to(s["out_dtype"])


def _ops():
    at = os.path.join(_ROOT, "torch-int_b200")
    if at not in sys.path:
        sys.path.insert(1, at)
    from torch_int import _CUDA
    return _CUDA


def run(s):
    if own:
        ops = _ops()
        if s["op"] == "append":
            q8 = ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["block_table"], s["query_starts"],
                                  s["kv_lens"], max_query_len=s["max_query_len"], q=s["q"], k_alpha=s["alpha"]["k"],
                                  v_alpha=s["alpha"]["v"], q_alpha=s["alpha"]["q"], rotary=s["rotary"],
                                  interleaved=s["interleaved"])
            return {"q": q8, "k": s["k_pages"], "v": s["v_pages"]}
        ctx = ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["query_starts"], s["kv_lens"],
                                  alpha_qk=s["alpha_qk"], alpha_pv=s["alpha_pv"], max_query_len=s["max_query_len"],
                                  max_kv_len=s["max_kv_len"], out_dtype=s["out_dtype"])
        return ctx.to(torch.float16) if ctx.dtype == torch.int8 else ctx
    return _append_plain(s) if s["op"] == "append" else _attention_plain(s)


def exact(case, seed):
    if case["op"] == "append" or case["out"] == "int8":
        return None  # whole numbers; a context rounded to whole units
    s = prepare(case, seed)
    new, keys = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    outs, start = [], 0
    for b, (t, n) in enumerate(zip(new, keys)):
        ids = s["block_table"][b, :-(-n // case["page"])].long()
        per_head = []
        for h in range(case["kv_heads"]):
            k = s["k_pages"][ids, h].reshape(-1, case["dim"])[:n].double()
            v = s["v_pages"][ids, h].reshape(-1, case["dim"])[:n].double()
            q = s["q"][start:start + t, h * group:(h + 1) * group].double().transpose(0, 1)  # [G, T, D]
            z = torch.matmul(q, k.t()).mul_(s["alpha_qk"])
            last = torch.arange(n - t, n, device="cuda")
            z.masked_fill_(torch.arange(n, device="cuda")[None, :] > last[:, None], float("-inf"))
            per_head.append(torch.matmul(torch.softmax(z, dim=-1), v).transpose(0, 1))
        outs.append(torch.cat(per_head, dim=1) * s["alpha_pv"])
        start += t
    return torch.cat(outs)


def work(case):
    new, keys = _lengths(case)
    tokens, dim, heads, kv_heads = sum(new), case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "append":
        values = tokens * (heads + 2 * kv_heads) * dim
        rotated = tokens * (heads + kv_heads) * case["rotary_dim"]
        places = len({n - t + i for t, n in zip(new, keys) for i in range(t)})
        return {"bytes": values * (_SIZES[case["dtype"]] + 1) + places * case["rotary_dim"] * 4, "flops": 3 * rotated + values}
    pairs = sum(t * (n - t) + t * (t + 1) // 2 for t, n in zip(new, keys))
    out = 1 if case["out"] == "int8" else 2
    return {"bytes": 2 * sum(keys) * kv_heads * dim + tokens * heads * dim * (1 + out), "flops": 4 * pairs * heads * dim}
