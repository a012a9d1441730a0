"""Keys and values in 4 bits, and attention over them, in 64-bit arithmetic on the CPU: what the kernels are held to.

A group is 16 neighbouring elements of a head of one token.  Its scale s is the number nearest to min(max |x|, 3360) / 7 among the
multiples of 2^-14 below 2^-11 and the numbers of four significant bits above; an element is c s with the whole number c nearest to
x / s, at most 7 in magnitude.  A group that holds a number that is not finite is NaN throughout."""
import torch

GROUP = 16


def scale_of_byte(b):
    b = b.to(torch.int64)
    e, f = b >> 3, (b & 7).double()
    s = torch.where(e == 0, f * 2.0 ** -14, (1.0 + f / 8.0) * torch.exp2(e.double() - 12.0))
    return torch.where(e == 31, torch.full_like(s, float("nan")), s)


def byte_of(x):
    """The scales' bytes of groups x [..., 16] (float64)."""
    table = scale_of_byte(torch.arange(168))
    most = x.abs().amax(-1)
    wanted = (most / 7.0).clamp(max=480.0).nan_to_num(0.0)
    near = (wanted[..., None] - table).abs()
    low = near.amin(-1, keepdim=True)
    tied = near == low                                   # two at most; the even byte is the even fraction
    index = torch.arange(168)
    pick = torch.where(tied & (index % 2 == 0), index, torch.where(tied, index + 1000, 5000)).amin(-1)
    pick = torch.where(pick >= 1000, pick - 1000, pick)
    return torch.where(most.isfinite(), pick, torch.full_like(pick, 255)).to(torch.uint8)


def quantised(x):
    """(codes c [..., d] as int64, scale bytes [..., d / 16]) of x [..., d]."""
    g = x.double().unflatten(-1, (-1, GROUP))
    b = byte_of(g)
    s = scale_of_byte(b)[..., None]
    c = torch.where(s > 0, torch.round(g / s), torch.zeros_like(g)).clamp(-7, 7)
    return c.nan_to_num(0.0).to(torch.int64).flatten(-2), b


def pack(c):
    u = (c + 8).to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def values(codes, scales):
    """float64 [..., d] of codes [..., d / 2] and scales [..., d / 16] (bytes)."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double() - 8.0
    return (c.unflatten(-1, (-1, GROUP)) * scale_of_byte(scales)[..., None]).flatten(-2)


def prepared(qkv, pos, nq, nkv, d, inv_freq, rot, q_gain, k_gain, eps):
    """(q, k, v) [rows, heads, d] in float64 after head norms and rotation."""
    x = qkv.double().unflatten(-1, (nq + 2 * nkv, d))
    out = []
    for heads, gain in ((x[:, :nq], q_gain), (x[:, nq:nq + nkv], k_gain)):
        if gain is not None:
            heads = heads / (heads.square().mean(-1, keepdim=True) + eps).sqrt() * gain.double()
        a = pos.double()[:, None, None] * inv_freq.double()
        u, w = heads[..., :rot // 2], heads[..., rot // 2:rot]
        out.append(torch.cat([u * a.cos() - w * a.sin(), w * a.cos() + u * a.sin(), heads[..., rot:]], -1))
    return out[0], out[1], x[:, nq + nkv:]


def gathered(part, table, slot, keys, page):
    """float64 [keys, heads, d] of a slot's positions 0 .. keys - 1."""
    pages = table[slot, :(keys + page - 1) // page].long()
    return values(part.codes[pages], part.scales[pages]).transpose(1, 2).flatten(0, 1)[:keys]


def attention(q, k, v, pos, window, scale, group):
    """(o, sum of p |v|, largest sum of |q| |k| scale) of queries q [heads, d] at ``pos`` over k, v [keys, kv heads, d]."""
    lo = max(0, pos - window + 1) if window else 0
    k, v = (x[lo:pos + 1].repeat_interleave(group, 1) for x in (k, v))
    s = torch.einsum("hd,khd->hk", q.double(), k) * scale
    p = torch.softmax(s, -1)
    reach = torch.einsum("hd,khd->hk", q.double().abs(), k.abs()).amax(-1) * abs(scale)
    return torch.einsum("hk,khd->hd", p, v), torch.einsum("hk,khd->hd", p, v.abs()), reach
