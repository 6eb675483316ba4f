"""Plain restatement of the KV-cache operators in 64 bits (test infrastructure): placement, rotation, quantisation,
read-back and attention over a 4-bit cache, row by row.  The reference has no counterpart (parity unpinned): the
definitions are those of include/aclnn_append_kv_cache.h, aclnn_gather_kv_cache.h and aclnn_paged_attention_int4.h."""
import math

import torch

F64 = torch.float64
END = torch.iinfo(torch.int32).max


def tokens(table, seq_len, query_start, T, bs, n_blocks):
    """For every row of a call: (sequence or -1, position or -1, page or -1, row in page)."""
    B = seq_len.shape[0]
    start = list(range(B + 1)) if query_start is None else query_start.tolist()
    out = [(-1, -1, -1, 0)] * T
    for b in range(B):
        n = start[b + 1] - start[b]
        for i in range(n):
            t, pos = start[b] + i, int(seq_len[b]) - n + i
            if t >= T:
                continue
            if not 0 <= pos < table.shape[1] * bs:
                out[t] = (b, -1, -1, 0)
                continue
            page = int(table[b, pos // bs])
            out[t] = (b, pos, page if 0 <= page < n_blocks else -1, pos % bs)
    return out


def rotate(x, table_row, interleaved):
    """x [heads, D], table_row [R]: cosines then sines."""
    x = x.to(F64).clone()
    R = table_row.shape[0]
    c, s = table_row[:R // 2].to(F64), table_row[R // 2:].to(F64)
    a, b = (torch.arange(0, R, 2), torch.arange(1, R, 2)) if interleaved else (torch.arange(R // 2), torch.arange(R // 2, R))
    u, v = x[:, a].clone(), x[:, b].clone()
    x[:, a], x[:, b] = u * c - v * s, v * c + u * s
    return x


def params4(x):
    """(scale, zero) float16 of rows x [..., D] (float64 input)."""
    lo, hi = x.amin(-1), x.amax(-1)
    s = ((hi - lo) / 15).clamp(max=65504.0).to(torch.float16)
    z = lo.clamp(-65504.0, 65504.0).to(torch.float16)
    return s, z


def unpack_k(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def unpack_v(codes):
    """[..., bs / 4, D / 2, 4] -> [..., bs, D]"""
    return unpack_k(codes.transpose(-1, -2)).flatten(-3, -2)


def pack_k(c):
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)


def pack_v(c):
    """[..., bs, D] -> [..., bs / 4, D / 2, 4]"""
    b = pack_k(c)
    return b.unflatten(-2, (-1, 4)).transpose(-1, -2).contiguous()


def values4(codes, params):
    """codes [blocks, Hkv, bs, D], params [blocks, Hkv, bs, 2] -> float64"""
    return codes.to(F64) * params[..., :1].to(F64) + params[..., 1:].to(F64)


def attention(q, k, v, table, seq_len, scale, Hkv, bs, query_start=None, causal=True, lists=None):
    """q [T, Hq, D]; k, v float64 pages [blocks, Hkv, bs, D].  Returns (out [T, Hq, D], lse [T, Hq], bound-helpers) with rows
    in no sequence NaN: (out, lse, spread) where spread[t, h] = (largest |V| seen, largest V span, largest sum |q| |K|)."""
    T, Hq, D = q.shape
    G, n_blocks = Hq // Hkv, k.shape[0]
    out = torch.full((T, Hq, D), float("nan"), dtype=F64)
    lse = torch.full((T, Hq), float("nan"), dtype=F64)
    big = torch.zeros((T, Hq, 2), dtype=F64)
    B = seq_len.shape[0]
    start = list(range(B + 1)) if query_start is None else query_start.tolist()
    cap = table.shape[1] * bs
    for b in range(B):
        n, length = start[b + 1] - start[b], max(int(seq_len[b]), 0)
        upto = min(length, cap)
        phys = [int(x) for x in table[b, :-(-upto // bs)]] if upto else []
        ok = torch.tensor([0 <= x < n_blocks for x in phys], dtype=torch.bool)
        idx = torch.tensor([x if 0 <= x < n_blocks else 0 for x in phys], dtype=torch.long)
        kb = k[idx].transpose(0, 1).reshape(Hkv, -1, D)[:, :upto] if upto else None
        vb = v[idx].transpose(0, 1).reshape(Hkv, -1, D)[:, :upto] if upto else None
        there = ok.repeat_interleave(bs)[:upto] if upto else None
        for i in range(n):
            t = start[b] + i
            if t >= T:
                continue
            see = min(upto, max(0, length - n + i + 1)) if causal else upto
            for h in range(Hq):
                if lists is None:
                    toks = torch.arange(see)[there[:see]] if see else torch.empty(0, dtype=torch.long)
                else:
                    row = lists[b, h if lists.shape[1] == Hq else h // G].tolist()
                    toks = []
                    for lp in row:
                        if not 0 <= lp < table.shape[1]:
                            break
                        toks += [x for x in range(lp * bs, (lp + 1) * bs) if x < see and bool(there[x])]
                    toks = torch.tensor(toks, dtype=torch.long)
                if len(toks) == 0:
                    out[t, h], lse[t, h] = 0.0, -3.4e38
                    continue
                kk, vv, qq = kb[h // G][toks], vb[h // G][toks], q[t, h].to(F64)
                e = (kk @ qq) * scale
                out[t, h] = torch.softmax(e, 0) @ vv
                lse[t, h] = torch.logsumexp(e, 0)
                big[t, h, 0] = vv.abs().max()
                big[t, h, 1] = (kk.abs().max() * 3 * qq.abs().sum()) * abs(scale)
    return out, lse, big


def attention_bound(out, big, D, out_dtype):
    """What the rounding of the operator may amount to, entry by entry.
      * a score is a sum of D exact products (11-bit q elements x codes, all exact in fp32) accumulated in fp32, times the
        scale, plus the zero's part: at most (D + 8) roundings of 2^-24 of the sum of magnitudes; with |K| <= kmax a code
        times its scale is at most 2 kmax and the zero at most kmax, so that sum is at most 3 kmax sum|q| scale =: A;
        exp2 and the reference's subtraction add 2^-21 (1 + A): delta = 2^-24 (D + 8) A + 2^-21 (1 + A);
      * a probability off by a relative delta moves numerator and denominator: 2 delta vmax;
      * p * s' is rounded to float16, half a step 2^-11 relative (and 2^-31 of the peak absolutely), times a code: the
        codes' part of a value is at most 2 vmax: 2^-11 * 2 vmax;
      * fp32 sums over the tokens, blockwise: 2^-20 vmax; the result is rounded once: eps / 2 of the output's type."""
    vmax, A = big[..., :1], big[..., 1:]
    delta = 2.0 ** -24 * (D + 8) * A + 2.0 ** -21 * (1 + A)
    half = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[out_dtype]
    return 2 * delta * vmax + 2.0 ** -10 * vmax + 2.0 ** -20 * vmax + half * out.abs() + 2.0 ** -24
