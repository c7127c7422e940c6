"""Plain 64-bit implementations of the quantised decoder-layer operators, on the CPU, with error bounds for the kernels.

A rounding to a type is off by at most eps / 2 of the value (U below); an fp32 operation by 2^-24 of its result. Each
function that returns a bound says which roundings it counts."""
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}  # half a step among the subnormal numbers
F32 = 2.0 ** -24


def decode(codes, params):
    """codes uint8 [..., D / 2], params [..., 2] -> float64 [..., D]."""
    out = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64)
    scale, mid = params[..., 0:1].double(), params[..., 1:2].double()
    out[..., 0::2] = mid + ((codes & 15).double() - 7.5) * scale
    out[..., 1::2] = mid + ((codes >> 4).double() - 7.5) * scale
    return out


def token_rows(cache, block, place):
    """(key codes, value codes [n, G, D / 2], key params, value params [n, G, 2]) of the slots (block[i], place[i])."""
    kc, vc, kp, vp = (t.cpu() for t in cache)
    return kc[block, :, place], vc[block, :, :, place], kp[block, :, place], vp[block, :, place]


def sequence_rows(cache, table, n, block_size):
    """The first n positions of a sequence, whose pages must all be in the pool, as token_rows()."""
    pos = torch.arange(n)
    return token_rows(cache, table.cpu().long()[pos // block_size], pos % block_size)


def attention(query, cache, tables, lens, qk_scale, tokens, block_size, mask=None, num_blocks=None):
    """(output, bound) float64 [batch * tokens, H, D] of paged_attention_int4, position by position of its definition.

    The bound counts: the output's rounding (U); the weights' rounding to bf16 (2^-8 of what they multiply, or 2^-16 for
    fp16 models, which keep the remainder), the fp32 sums over codes offset by 23.5, and the scores' fp32 errors, which
    change a weight by their size."""
    dtype = query.dtype
    q = query.cpu().double()
    rows, h, d = q.shape
    num_blocks = cache[0].shape[0] if num_blocks is None else num_blocks
    g = cache[0].shape[1]
    group = h // g
    out = torch.zeros((rows, h, d), dtype=torch.float64)
    bound = torch.zeros_like(out)
    tables, lens = tables.cpu(), lens.cpu()
    reach = tables.shape[1] * block_size
    m = None if mask is None else mask.cpu().double()
    for b in range(tables.shape[0]):
        n = min(max(int(lens[b]), 0), reach)
        if n == 0:
            continue
        pos = torch.arange(n)
        page = tables[b].long()[pos // block_size]
        there = (page >= 0) & (page < num_blocks)
        kc, vc, kp, vp = token_rows(cache, torch.where(there, page, 0), pos % block_size)
        k, v = decode(kc, kp), decode(vc, vp)  # [n, g, d]
        ks, km = kp[..., 0].double(), kp[..., 1].double()
        vs, vm = vp[..., 0].double(), vp[..., 1].double()
        for j in range(tokens):
            seen = n - tokens + 1 + j
            for head in range(h):
                kv = head // group
                s = k[:, kv] @ q[b * tokens + j, head] * qk_scale
                hide = ~there | (pos >= seen)
                if m is not None:
                    row = m[b if m.shape[0] > 1 else 0, head if m.shape[1] > 1 else 0, j if m.shape[2] > 1 else 0]
                    bias = torch.full((n,), -torch.inf, dtype=torch.float64)
                    bias[: min(n, len(row))] = row[: min(n, len(row))]
                    hide |= bias == -torch.inf
                    s = s + torch.where(hide, 0.0, bias)
                s = torch.where(hide, -torch.inf, s)
                top = s.max()
                if top == -torch.inf:
                    continue
                w = torch.where(hide, 0.0, torch.exp(s - top))
                w = w / w.sum()
                live = ~hide
                o = (w[live, None] * v[live, kv]).sum(0)
                out[b * tokens + j, head] = o
                # fp32 in a score: sums of D terms (offset codes up to 40 times the scale, the middle), then a few more
                sum_q = q[b * tokens + j, head].abs().sum()
                err = F32 * (2 * (d + 8) * (40.0 * ks[live, kv] + km[live, kv].abs()) * sum_q * qk_scale)
                # (a mask of the type's lowest value leaves scores that differ by less than their last bit: no error in
                # the differences that the weights are made of; the weights of others beside such scores are 0)
                size = torch.where(s[live].abs() < 1e30, s[live].abs(), 0.0)
                err = float((err + 8 * F32 * size).max()) + 8 * F32
                vl, wl = v[live, kv], w[live]
                spread = (wl[:, None] * (vl - vm[live, kv][:, None]).abs()).sum(0)
                p_err = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -16
                sums = F32 * (n / 32 + 96) * ((wl * vs[live, kv]).sum() * 40.0 + (wl * vm[live, kv].abs()).sum())
                bound[b * tokens + j, head] = (U[dtype] * o.abs() + p_err * spread + 2 * err * (wl[:, None] * vl.abs()).sum(0) +
                                               sums + TINY[dtype]) * 1.01
    return out, bound


def quantised_row_ok(x, codes, params):
    """Whether 4-bit rows (codes uint8 [..., D / 2], params [..., 2]) are what the definition makes of x [..., D]: the params
    within their type's rounding (and fp32's before it), each code nearest to its place under the stored params."""
    dtype = x.dtype
    v = x.double()
    hi, lo = v.amax(-1), v.amin(-1)
    finite = torch.isfinite(v).all(-1)
    scale, mid = params[..., 0].double(), params[..., 1].double()
    ok = ~finite & scale.isnan() & mid.isnan()
    want_s, want_m = (hi - lo) / 15.0, (hi + lo) / 2.0
    floor = 2.0 ** -126 if dtype == torch.bfloat16 else TINY[dtype]  # bf16 scales below the normal numbers are 0
    good = (scale - want_s).abs() <= want_s * (U[dtype] + 4 * F32) + floor
    good &= (mid - want_m).abs() <= want_m.abs() * (U[dtype] + 2 * F32) + 2 * F32 * torch.maximum(hi.abs(), lo.abs()) + TINY[dtype]
    c = torch.empty(v.shape, dtype=torch.float64)
    c[..., 0::2], c[..., 1::2] = (codes & 15).double(), (codes >> 4).double()
    place = ((v - mid[..., None]) / scale.clamp_min(1e-300)[..., None] + 7.5).clamp(0, 15)
    near = (c - place).abs() <= 0.5 + 64 * F32 * 16  # fp32: the difference, the reciprocal, the sum
    tie = (place - place.floor() == 0.5) & ((v - mid[..., None]).float().double() == v - mid[..., None])
    near = (near & (~tie | (c == place.round()))).all(-1)  # exact ties, common with so few bits, go to the even code
    good &= torch.where(scale == 0, (c == 8).all(-1), near)
    return bool((ok | (finite & good)).all())


def norm_quant_ok(x, residual, gamma, eps, codes, scale, residual_out):
    """Whether rms_norm_quant's outputs are what the definition makes of its inputs (finite rows)."""
    dtype = x.dtype
    s = x.float() if residual is None else x.float() + residual.float()
    s = s.to(dtype)
    if residual is not None and not torch.equal(residual_out, s):
        return False
    s = s.double()
    sg = s * gamma.double()
    dim = s.shape[-1]
    want = sg.abs().amax(-1) / torch.sqrt((s * s).mean(-1) + eps) / 127.0
    # a sum of dim squares, whatever its order, then a square root, a reciprocal and three products
    if not bool(((scale.double() - want).abs() <= want * F32 * (dim / 2 + 12) + 1e-45).all()):
        return False
    most = sg.abs().amax(-1, keepdim=True)
    place = torch.where(most > 0, sg / most.clamp_min(1e-300) * 127.0, 0.0)
    return bool(((codes.double() - place).abs() <= 0.5 + 127 * 6 * F32).all())


def linear(x, w, x_scale, w_scale, bias, dtype):
    """(output, bound) float64: the integer sum is exact; its conversion, two products, the bias and the final rounding."""
    total = x.double() @ w.double().t()
    value = total * x_scale.double()[:, None] * w_scale.double()
    more = 0.0 if bias is None else bias.double()
    out = value + more
    size = value.abs() + (0.0 if bias is None else bias.double().abs())
    return out, U[dtype] * out.abs() + 6 * F32 * size + TINY[dtype]
