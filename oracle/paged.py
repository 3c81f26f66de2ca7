"""Plain 64-bit restatement of the paged int8 cache operators (test infrastructure).

Formulas only: a Python loop over sequences and tokens' positions, dense products in float64.
"""
import torch


def paged_positions(query_starts, kv_lens):
    """[(sequence, first token, new tokens, keys)] from the index arrays."""
    qs, kl = [int(x) for x in query_starts], [int(x) for x in kv_lens]
    return [(b, qs[b], qs[b + 1] - qs[b], kl[b]) for b in range(len(kl))]


def rotate(x, table, interleaved):
    """x [T, H, D] fp32, table [T, rd] fp32 (cosines, sines): every product and sum rounded to fp32."""
    rd = table.shape[-1]
    c, s = table[:, None, :rd // 2], table[:, None, rd // 2:]
    y = x.clone()
    if interleaved:
        x1, x2 = x[..., 0:rd:2], x[..., 1:rd:2]
        y[..., 0:rd:2], y[..., 1:rd:2] = x1 * c - x2 * s, x2 * c + x1 * s
    else:
        x1, x2 = x[..., :rd // 2], x[..., rd // 2:rd]
        y[..., :rd // 2], y[..., rd // 2:rd] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


def quantise(x, alpha):
    """int8 = sat_rne(alpha * x); NaN gives 0."""
    return torch.nan_to_num((x * alpha).round(), nan=0.0, posinf=127.0, neginf=-128.0).clamp(-128, 127).to(torch.int8)


def paged_append(k, v, k_pages, v_pages, block_table, query_starts, kv_lens, q=None, k_alpha=1.0, v_alpha=1.0,
                 q_alpha=1.0, rotary=None, interleaved=False):
    """Writes into k_pages / v_pages (CPU tensors); returns the int8 queries or None."""
    page_size = k_pages.shape[2]
    out = None if q is None else torch.zeros(q.shape, dtype=torch.int8)
    for b, q0, t, keys in paged_positions(query_starts, kv_lens):
        pos = torch.arange(keys - t, keys)
        ks, vs = k[q0:q0 + t].float(), v[q0:q0 + t].float()
        table = None if rotary is None else rotary[pos]
        if table is not None:
            ks = rotate(ks, table, interleaved)
        pages = block_table[b][(pos // page_size).long()].long()
        k_pages[pages, :, (pos % page_size).long()] = quantise(ks, k_alpha)
        v_pages[pages, :, (pos % page_size).long()] = quantise(vs, v_alpha)
        if q is not None:
            x = q[q0:q0 + t].float()
            out[q0:q0 + t] = quantise(x if table is None else rotate(x, table, interleaved), q_alpha)
    return out


def paged_attention(q, k_pages, v_pages, block_table, query_starts, kv_lens, alpha_qk, alpha_pv):
    """(context, spread) in float64 [N, Hq, D]: spread = |alpha_pv| * sum_j softmax_j * |v_j|, the scale that relative
    errors of the probabilities act on.  Rows that see no key and rows of no sequence are 0."""
    n, hq, d = q.shape
    hkv = k_pages.shape[1]
    group = hq // hkv
    ctx = torch.zeros((n, hq, d), dtype=torch.float64)
    spread = torch.zeros_like(ctx)
    for b, q0, t, keys in paged_positions(query_starts, kv_lens):
        if t == 0 or keys == 0:
            continue
        page_size = k_pages.shape[2]
        ids = block_table[b, :-(-keys // page_size)].long()
        ks = k_pages[ids].transpose(0, 1).reshape(hkv, -1, d)[:, :keys].double()
        vs = v_pages[ids].transpose(0, 1).reshape(hkv, -1, d)[:, :keys].double()
        x = q[q0:q0 + t].double().view(t, hkv, group, d).permute(1, 2, 0, 3)          # [Hkv, G, T, D]
        s = (x @ ks[:, None].transpose(2, 3)) * alpha_qk
        seen = torch.arange(keys)[None, :] <= torch.arange(keys - t, keys)[:, None]   # [T, S]
        s = s.masked_fill(~seen, float("-inf"))
        p = torch.nan_to_num(torch.softmax(s, dim=-1), nan=0.0)                       # no key: softmax of nothing
        for dst, val in ((ctx, vs), (spread, vs.abs())):
            y = (p @ val[:, None]).permute(2, 0, 1, 3).reshape(t, hq, d)
            dst[q0:q0 + t] = y * (alpha_pv if dst is ctx else abs(alpha_pv))
    return ctx, spread


def model_attention(sd, prefix, hidden_int8, mask, num_heads, past=None, trace=None):
    """attention() of opt_model.py as the paged model path computes it: probabilities kept in 64 bits, not rounded to units
    of 1/127, so the scale of pv_bmm, which counts those units, is taken 127 times; one rounding of the context to int8."""
    from . import opt_model as OM
    bsz, tgt, e = hidden_int8.shape
    d = e // num_heads
    x2d = hidden_int8.reshape(-1, e)
    q, k, v = (OM._linear_s8(sd, f"{prefix}.{n}", x2d).view(bsz, tgt, num_heads, d).transpose(1, 2) for n in ("q_proj", "k_proj", "v_proj"))
    if past is not None:
        k, v = torch.cat([past[0], k], dim=2), torch.cat([past[1], v], dim=2)
    scores = (q.double() @ k.double().transpose(2, 3)) * OM._f(sd, prefix + ".qk_bmm.a")
    p = torch.softmax(scores.masked_fill(mask < 0, float("-inf")), dim=-1)
    ctx = (127.0 * OM._f(sd, prefix + ".pv_bmm.a") * (p @ v.double())).round().clamp(-128, 127).to(torch.int8)
    ctx = ctx.transpose(1, 2).reshape(bsz * tgt, e).contiguous()
    return OM._linear_f32(sd, prefix + ".out_proj", ctx).view(bsz, tgt, e), (k, v)
