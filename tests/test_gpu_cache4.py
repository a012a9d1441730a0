"""The cache in 4 bits on the device: appending (head norms, rotation, codes), reading back, and attention over it, against 64-bit
arithmetic on the CPU.  Bytes of the pools that nothing has written are 0xff, which reads as NaN: a kernel that lets a key count
that its row does not see shows it."""
import math
import random

import pytest
import torch

import citlali_b200 as cb
import plain_cache4 as plain
from citlali_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Step:
    """A cache of `slots` sequences in shuffled pages, and a step of rows at the end of them."""

    def __init__(self, past, new, nkv, d, page=64, seed=0, slots=None, spare_pages=3):
        rng = random.Random(seed)
        self.past, self.new, self.page, self.nkv, self.d = list(past), list(new), page, nkv, d
        slots = slots or len(past) + 2
        self.slots = rng.sample(range(slots), len(past))
        need = [(p + n + page - 1) // page for p, n in zip(past, new)]
        pages = sum(need) + spare_pages
        order = rng.sample(range(pages), pages)
        self.table = torch.zeros(slots, max(need) + 1, dtype=torch.int32)
        for s, n in zip(self.slots, need):
            self.table[s, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        ff = lambda w: torch.full((pages, nkv, page, w), 255, dtype=torch.uint8)
        self.keys, self.values = (cb.Packed4(ff(d // 2), ff(d // 16)) for _ in range(2))
        self.row_slot = [s for s, n in zip(self.slots, new) for _ in range(n)]
        self.row_pos = [p + i for p, n in zip(past, new) for i in range(n)]
        self.window = None

    def fill(self, seed, tokens=None):
        """Random keys and values for all positions, past and new."""
        g = torch.Generator().manual_seed(seed)
        for part in (self.keys, self.values):
            for s, p, n in zip(self.slots, self.past, self.new):
                x = torch.randn(p + n, self.nkv, self.d, generator=g).bfloat16()
                c, b = plain.quantised(x)
                for at in range(p + n):
                    page, place = int(self.table[s, at // self.page]), at % self.page
                    part.codes[page, :, place] = plain.pack(c[at])
                    part.scales[page, :, place] = b[at]

    def view(self):
        dev = lambda part: cb.Packed4(part.codes.to(DEV), part.scales.to(DEV))
        return cb.KVView(dev(self.keys), dev(self.values), self.table.to(DEV), self.page,
                         cb.KVRequirement(self.nkv, self.d, self.window, packed4=True))

    def batch(self):
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        start = [0]
        for n in self.new:
            start.append(start[-1] + n)
        return cb.StepBatch(ints([0] * len(self.row_slot)), ints(self.row_slot), ints(self.row_pos), ints(start), ints(self.slots),
                            ints(self.past), ints([]), slots=list(self.slots), past=list(self.past), n_new=list(self.new))


def gains(d, g, dtype, on):
    return [(1 + 0.3 * torch.randn(d, generator=g)).to(dtype) if on else None for _ in range(2)]


def freqs(rot, theta=1e4):
    return torch.pow(torch.tensor(theta, dtype=torch.float64), -2.0 * torch.arange(rot // 2, dtype=torch.float64) / max(rot, 1)).float()


def on_device(*tensors):
    return [None if t is None else t.to(DEV) for t in tensors]


APPEND = [
    # nq, nkv, d, rotated, head norms, rows' dtype, gains' dtype, page, past, new
    (16, 8, 128, 128, True, torch.bfloat16, torch.bfloat16, 64, [63, 0, 130], [1, 1, 1]),
    (4, 2, 128, 64, True, torch.bfloat16, torch.float32, 64, [5], [131]),
    (3, 1, 64, 64, False, torch.bfloat16, torch.bfloat16, 64, [0, 70], [65, 7]),
    (2, 2, 256, 256, True, torch.float32, torch.float32, 64, [1], [3]),
    (10, 2, 80, 40, False, torch.float32, torch.float32, 64, [60, 0], [9, 33]),
    (6, 3, 48, 48, True, torch.bfloat16, torch.float32, 7, [3, 20], [5, 1]),
    (1, 1, 16, 6, True, torch.float32, torch.bfloat16, 16, [0], [40]),
    (2, 1, 96, 0, True, torch.bfloat16, torch.bfloat16, 64, [0], [5]),
    (16, 8, 128, 128, True, torch.bfloat16, torch.bfloat16, 64, [0], [700]),
    (3, 3, 32, 32, True, torch.float32, torch.float32, 64, [100000], [2]),
]


@pytest.mark.parametrize("nq,nkv,d,rot,norms,dtype,gain_dtype,page,past,new", APPEND)
@pytest.mark.parametrize("in_place", [False, True])
def test_append(nq, nkv, d, rot, norms, dtype, gain_dtype, page, past, new, in_place):
    g = torch.Generator().manual_seed(nq * 1000 + d + rot)
    st = Step(past, new, nkv, d, page, seed=d)
    rows = len(st.row_slot)
    qkv = (torch.randn(rows, (nq + 2 * nkv) * d, generator=g) * torch.exp(torch.randn((nq + 2 * nkv) * d, generator=g))).to(dtype)
    q_gain, k_gain = gains(d, g, gain_dtype, norms)
    inv_freq = freqs(rot)
    kv = st.view()
    before = [p.clone() for part in (kv.keys, kv.values) for p in (part.codes, part.scales)]
    slot, pos = (torch.tensor(v, dtype=torch.int32) for v in (st.row_slot, st.row_pos))
    dev, qg, kg, f, s, p = on_device(qkv.clone(), q_gain, k_gain, inv_freq, slot, pos)
    q_out = None if in_place else torch.full((rows, nq * d), 7.0, dtype=dtype, device=DEV)
    ops.cache4_append(dev, kv, s, p, nq, nkv, d, f, rot, qg, kg, 1e-6, q_out=q_out)
    got_q = (dev[:, :nq * d] if in_place else q_out).cpu().double().unflatten(-1, (nq, d))
    assert torch.equal(dev[:, nq * d:].cpu(), qkv[:, nq * d:])
    if not in_place:
        assert torch.equal(dev.cpu(), qkv)
    q, k, v = plain.prepared(qkv, pos, nq, nkv, d, inv_freq, rot, q_gain, k_gain, 1e-6)
    # queries: the norm's sum, root, two products (2^-21 with room), the turn's products and sum against the pair's size, one rounding
    pair = q.abs().clone()
    pair[..., :rot // 2] = pair[..., rot // 2:rot] = (q[..., :rot // 2].square() + q[..., rot // 2:rot].square()).sqrt()
    tol = torch.finfo(dtype).eps / 2 * q.abs() + 2.0 ** -20 * pair + 1e-30
    assert ((got_q - q).abs() <= tol).all(), float(((got_q - q).abs() / tol).max())

    touched = [torch.zeros(t.shape[:3], dtype=torch.bool) for t in before[::2]]
    for part, want, mark in zip((kv.keys, kv.values), (k, v), touched):
        codes, scales = part.codes.cpu(), part.scales.cpu()
        for r in range(rows):
            page_id, place = int(st.table[st.row_slot[r], st.row_pos[r] // page]), st.row_pos[r] % page
            mark[page_id, :, place] = True
            have_c = torch.stack([codes[page_id, :, place] & 15, codes[page_id, :, place] >> 4], -1).flatten(-2).to(torch.int64) - 8
            have_b = scales[page_id, :, place]
            c, b = plain.quantised(want[r])
            x = want[r].unflatten(-1, (-1, 16))
            if want is v:                              # as they came: the same bytes in any precision where elements have 16 bits
                if dtype == torch.bfloat16:
                    assert torch.equal(have_b, b) and torch.equal(have_c, c)
                    continue
                slack = 2.0 ** -22                     # of float32 elements only the two divisions are rounded
            else:
                slack = 2.0 ** -19                     # as the queries above; a group's elements are within 2^10 of its largest
            # a byte that is another one: only where the largest element over 7 lies next to the middle of two scales
            wanted = (x.abs().amax(-1) / 7).clamp(max=480.0)
            s_have, s_want = plain.scale_of_byte(have_b), plain.scale_of_byte(b)
            assert ((s_have - wanted).abs() <= (s_want - wanted).abs() + 2 * slack * wanted + 1e-30).all()
            # a code that is not the nearest one: only next to the middle of two
            assert have_c.min() >= -7 and have_c.max() <= 7
            t = torch.where(s_have[..., None] > 0, x / s_have[..., None], torch.zeros_like(x))
            off = (have_c.unflatten(-1, (-1, 16)).double() - t.clamp(-7, 7)).abs()
            assert (off <= 0.5 + slack * 16).all(), float(off.max())
    for t, was, mark in zip((kv.keys.codes, kv.keys.scales, kv.values.codes, kv.values.scales), before,
                            (touched[0], touched[0], touched[1], touched[1])):
        assert torch.equal(t.cpu()[~mark], was.cpu()[~mark])          # nothing else was written

    # what reading back gives are the codes' values
    if rows:
        keys, vals = ops.cache4_read(kv, s, p, dtype=torch.float32)
        keys16, vals16 = ops.cache4_read(kv, s, p)
        for part, out, out16 in ((kv.keys, keys, keys16), (kv.values, vals, vals16)):
            codes, scales = part.codes.cpu(), part.scales.cpu()
            want = torch.stack([plain.values(codes[int(st.table[a, b // page]), :, b % page], scales[int(st.table[a, b // page]), :, b % page])
                                for a, b in zip(st.row_slot, st.row_pos)])
            assert torch.equal(out.cpu().double(), want) and torch.equal(out16.cpu().double(), want)


def test_append_without_storing_and_other_row_pitches():
    g = torch.Generator().manual_seed(1)
    st = Step([10], [6], 2, 64)
    qkv = torch.randn(6, 4 * 64, generator=g).bfloat16()
    dev, f, s, p = on_device(qkv, freqs(64), torch.tensor(st.row_slot, dtype=torch.int32), torch.tensor(st.row_pos, dtype=torch.int32))
    # a layer that reads another layer's cache has queries only
    out = torch.zeros(6, 300, dtype=torch.bfloat16, device=DEV)[:, :256]
    ops.cache4_append(dev, None, s, p, 4, 0, 64, f, 64, q_out=out, store=False)
    q, _, _ = plain.prepared(qkv, torch.tensor(st.row_pos), 4, 0, 64, freqs(64), 64, None, None, 0.0)
    assert ((out.cpu().double().unflatten(-1, (4, 64)) - q).abs() <= 2.0 ** -8 * q.abs() + 2.0 ** -18 * 4).all()
    # the same rows with keys and values that are not stored
    kv = st.view()
    before = kv.keys.codes.clone()
    ops.cache4_append(dev, kv, s, p, 2, 1, 64, f, 64, q_out=torch.empty(6, 128, dtype=torch.bfloat16, device=DEV), store=False)
    assert torch.equal(kv.keys.codes, before)


def test_reading_what_is_not_there():
    st = Step([70, 3], [1, 1], 2, 64, slots=4)
    st.fill(3)
    view = st.view()
    view.page_table[st.slots[1], 1] = -1                 # names no page
    view.page_table[st.slots[1], 0] = view.keys.codes.shape[0]
    a, b, wide = st.slots[0], st.slots[1], view.page_table.shape[1] * 64
    slots = [a, a, a, -1, 4, 2 ** 31 - 1, b, b, a, a]
    positions = [0, -1, wide, 5, 5, 5, 64, 0, 2 ** 31 - 1, 70]
    for dtype in (torch.bfloat16, torch.float32):
        read = ops.cache4_read(view, *on_device(torch.tensor(slots, dtype=torch.int32), torch.tensor(positions, dtype=torch.int32)), dtype=dtype)
        for part, have in zip((st.keys, st.values), read):
            want = plain.gathered(part, st.table, a, 71, 64)
            assert torch.equal(have[[0, 9]].cpu().double(), want[[0, 70]]) and have[1:9].isnan().all()


def test_what_is_not_finite_stays_in_its_group():
    st = Step([0], [4], 1, 64)
    qkv = torch.zeros(4, 3 * 64)
    qkv[:, 64:] = torch.randn(4, 128, generator=torch.Generator().manual_seed(3))
    qkv[1, 64 + 20] = float("nan")
    qkv[2, 128 + 40] = float("inf")
    qkv[3, 128:144] = 0.0
    for dtype in (torch.float32, torch.bfloat16):
        kv = st.view()
        s, p = on_device(torch.tensor(st.row_slot, dtype=torch.int32), torch.tensor(st.row_pos, dtype=torch.int32))
        ops.cache4_append(qkv.to(dtype).to(DEV), kv, s, p, 1, 1, 64, freqs(0).to(DEV), 0)
        k, v = (t.cpu()[:, 0] for t in ops.cache4_read(kv, s, p))
        nan_k, nan_v = k.isnan(), v.isnan()
        assert nan_k.sum() == 16 and nan_k[1, 16:32].all()
        assert nan_v.sum() == 16 and nan_v[2, 32:48].all()
        assert (v[3, :16] == 0).all()


def test_large_and_tiny_numbers_are_held_at_the_ends_of_the_range():
    st = Step([0], [3], 1, 16)
    qkv = torch.zeros(3, 48)
    qkv[0, 32:] = 1e5 * torch.linspace(-1, 1, 16)
    qkv[1, 32:] = 1e-9
    qkv[2, 32:] = torch.linspace(-1, 1, 16) * 1e-3
    kv = st.view()
    s, p = on_device(torch.tensor(st.row_slot, dtype=torch.int32), torch.tensor(st.row_pos, dtype=torch.int32))
    ops.cache4_append(qkv.to(DEV), kv, s, p, 1, 1, 16, freqs(0).to(DEV), 0)
    v = ops.cache4_read(kv, s, p, dtype=torch.float32)[1].cpu()[:, 0]
    assert v[0].abs().max() == 3360.0 and (v[1] == 0).all()
    assert torch.equal(v.double(), plain.values(plain.pack(plain.quantised(qkv[:, 32:])[0]), plain.quantised(qkv[:, 32:])[1]))


# ---- attention --------------------------------------------------------------------------------------------------------------

def check_attention(st, nq, dtype, window, seed, out_rows=None, scale=None, expect_nan=None, way=("codes",)):
    """By the kernels that read codes: those for single tokens, or with ``way`` ("tiles", 0, tiles, cluster) the one for runs."""
    g = torch.Generator().manual_seed(seed)
    nkv, d, group = st.nkv, st.d, nq // st.nkv
    rows = len(st.row_slot)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    pitch = (nq + 2 * nkv) * d
    q = (1.5 * torch.randn(rows, pitch, generator=g)).to(dtype)
    out = torch.full((out_rows or rows, nq * d), 5.0, dtype=dtype, device=DEV)
    batch = st.batch()
    batch.runs4[nq, nkv, d, window, pitch] = way
    ops.cache4_attention(q.to(DEV), pitch, st.view(), batch, out, nq, nkv, d, window, scale)
    got = out.cpu().double()
    assert (got[rows:] == 5.0).all()
    row = 0
    for s, past, n in zip(st.slots, st.past, st.new):
        k, v = (plain.gathered(part, st.table, s, past + n, st.page) for part in (st.keys, st.values))
        for i in range(n):
            o, weight, reach = plain.attention(q[row, :nq * d].view(nq, d), k, v, past + i, window, scale, group)
            have = got[row].view(nq, d)
            # a score is a sum of d products in 32 bits (chains of d / 16 steps on the tensor cores): off by at most
            # (d / 8 + 8) 2^-23 of what its products add up to; twice that on a weight and on the weights' sum
            steps = d / 8 + 8 if dtype == torch.bfloat16 else d + 8
            off = 4 * steps * 2.0 ** -23 * reach[:, None]
            # the weights' roundings (half a step of a half, subnormal below 2^-25 of the largest; none in 32 bits), the sums', the result's
            off = off + (2.0 ** -11 if dtype == torch.bfloat16 else 0.0) + (past + n + 64) / 32 * 2.0 ** -23
            tol = torch.finfo(dtype).eps / 2 * o.abs() + off * weight
            if way[0] == "tiles":                        # (there a weight below 2^-20 of the largest is a subnormal half)
                tol = tol + (past + n) * 2.0 ** -31 * v.nan_to_num(0.0).abs().max()
            if expect_nan is not None and expect_nan(s, past + i):
                assert have.isnan().all()
            else:
                assert have.isfinite().all(), (s, past + i)
                assert ((have - o).abs() <= tol).all(), (s, past + i, float(((have - o).abs() / tol).max()))
            row += 1
    return got


DECODE = [
    # nq, nkv, d, lengths (with the new token), window
    (16, 8, 128, [1], 0),
    (16, 8, 128, [16, 17, 15, 64, 65, 63, 1, 2], 0),
    (2, 1, 128, [1000], 0),
    (40, 8, 128, [300, 1, 77, 2500], 0),
    (8, 1, 128, [129, 640], 100),
    (16, 1, 128, [129, 640], 64),
    (24, 2, 128, [70, 5], 0),
    (20, 1, 128, [333], 33),
    (4, 4, 64, [5, 900], 0),
    (12, 1, 64, [130, 16], 17),
    (6, 2, 256, [200, 3], 0),
    (5, 5, 128, [64] * 40, 0),
    (2, 2, 128, list(range(1, 80)), 0),
]


@pytest.mark.parametrize("nq,nkv,d,lengths,window", DECODE)
def test_single_tokens(nq, nkv, d, lengths, window):
    st = Step([n - 1 for n in lengths], [1] * len(lengths), nkv, d, seed=nq + d)
    st.fill(len(lengths))
    check_attention(st, nq, torch.bfloat16, window, nq, out_rows=len(lengths) + 2)


RUNS = [
    # nq, nkv, d, past, new, window
    (16, 8, 128, [0], [1 + 16], 0),
    (16, 8, 128, [0, 5, 100], [7, 1, 39], 0),
    (40, 8, 128, [61, 200], [24, 5], 50),
    (4, 4, 128, [0], [150], 0),
    (8, 1, 64, [33, 0], [20, 3], 16),
    (6, 2, 256, [10], [9], 0),
    (40, 2, 128, [17], [4], 0),
    (3, 1, 128, [1000, 3], [2, 70], 7),
]


@pytest.mark.parametrize("nq,nkv,d,past,new,window", RUNS)
def test_runs_of_tokens(nq, nkv, d, past, new, window):
    st = Step(past, new, nkv, d, seed=nq + d)
    st.fill(sum(new))
    check_attention(st, nq, torch.bfloat16, window, nq, out_rows=sum(new) + 1)


TILES = [
    # nq, nkv, d, past, new, window
    (16, 8, 128, [0], [17], 0),
    (16, 8, 128, [0, 5, 100], [7, 1, 39], 0),
    (40, 8, 128, [61, 200], [24, 5], 50),
    (4, 4, 128, [0], [150], 0),
    (8, 1, 64, [33, 0], [20, 3], 16),
    (40, 2, 128, [17], [4], 0),
    (3, 1, 128, [1000, 3], [2, 70], 7),
    (6, 2, 64, [700, 0, 64], [65, 128, 1], 0),
    (128, 1, 64, [100], [3], 0),
    (2, 1, 128, [640, 63], [129, 64], 64),
]


def tiles_of(nq, nkv, new):
    tokens = 128 // (nq // nkv)
    return nkv * sum(-(-n // tokens) for n in new)


@pytest.mark.parametrize("nq,nkv,d,past,new,window", TILES)
@pytest.mark.parametrize("cluster", [1, 2, 4, 8])
def test_runs_of_tokens_in_tiles(nq, nkv, d, past, new, window, cluster):
    st = Step(past, new, nkv, d, seed=nq + d)
    st.fill(sum(new))
    check_attention(st, nq, torch.bfloat16, window, nq, out_rows=sum(new) + 1, way=("tiles", 0, tiles_of(nq, nkv, new), cluster))


@pytest.mark.parametrize("nq,nkv,d,past,new,window,few", [
    (4, 2, 128, [300, 0, 77, 1000, 5, 64], [1, 90, 4, 1, 0, 5], 0, 4),
    (8, 1, 64, [10, 700, 0], [1, 1, 33], 50, 1),
    (5, 1, 128, [10, 70], [40, 1], 0, 1),
])
def test_short_and_long_runs_in_one_step(nq, nkv, d, past, new, window, few):
    """Sequences of up to ``few`` new tokens by the kernel for single tokens, the others in tiles: each row by one of them."""
    st = Step(past, new, nkv, d, seed=nq + d)
    st.fill(sum(new))
    before = ops.launch_count()
    check_attention(st, nq, torch.bfloat16, window, nq, out_rows=sum(new) + 1,
                    way=("tiles", few, tiles_of(nq, nkv, [n for n in new if n > few]), 2))
    assert ops.launch_count() - before == 2


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", ["keys", "values"])
@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("cluster", [1, 2])
def test_a_token_that_is_not_finite_in_tiles(d, which, window, cluster):
    st = Step([30, 10], [90, 50], 1, d, seed=5)
    st.fill(5)
    slot, at = st.slots[0], 75
    part = getattr(st, which)
    part.scales[int(st.table[slot, at // 64]), 0, at % 64, d // 16 - 1] = 255
    check_attention(st, 2, torch.bfloat16, window, 2, expect_nan=lambda s, p: s == slot and p >= at and (not window or p < at + window),
                    way=("tiles", 0, tiles_of(2, 1, st.new), cluster))


def test_tiles_whose_scores_spread_and_odd_queries():
    st = Step([500, 0, 63], [3, 70, 2], 2, 128, seed=9)
    st.fill(9)
    new = st.new
    for cluster in (1, 4):
        way = ("tiles", 0, tiles_of(4, 2, new), cluster)
        check_attention(st, 4, torch.bfloat16, 0, 3, scale=1.0, way=way)             # weights from 1 to 2^-200
        check_attention(st, 4, torch.bfloat16, 0, 4, scale=0.0, way=way)             # all keys alike
        q = torch.randn(75, 4 * 128, generator=torch.Generator().manual_seed(1)).bfloat16()
        outs = []
        stream = torch.cuda.Stream()
        for up in (1.0, 2.0 ** 60, 2.0 ** -60, 1.0):
            given, view, batch = (q * up).to(DEV), st.view(), st.batch()
            batch.runs4[4, 2, 128, 0, 512] = way
            out = torch.empty(75, 4 * 128, dtype=torch.bfloat16, device=DEV)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                ops.cache4_attention(given, 512, view, batch, out, 4, 2, 128, 0, 0.1 / up)
            stream.synchronize()
            outs.append(out)
        assert all(torch.equal(outs[0], o) for o in outs[1:])
        odd = q.clone()
        odd[4] = 0.0
        odd[5, 3] = float("nan")
        odd[6, 130] = float("inf")
        batch = st.batch()
        batch.runs4[4, 2, 128, 0, 512] = way
        out = torch.empty(75, 4 * 128, dtype=torch.bfloat16, device=DEV)
        ops.cache4_attention(odd.to(DEV), 512, st.view(), batch, out, 4, 2, 128, 0, 0.1)
        got, plainly = out.cpu().view(75, 4, 128), outs[0].cpu().view(75, 4, 128)
        assert got[5, 0].isnan().all() and not got[6, 1].isfinite().any()
        alike = torch.ones(75, 4, dtype=torch.bool)
        alike[4] = alike[5, 0] = alike[6, 1] = False
        assert torch.equal(got[alike], plainly[alike])
        v = plain.gathered(st.values, st.table, st.slots[1], 2, 64).mean(0)          # row 4 is the second token of its sequence
        assert ((got[4].double() - v.repeat_interleave(2, 0)).abs() <= 2.0 ** -8 * v.abs().max() + 2.0 ** -10).all()


@pytest.mark.parametrize("nq,nkv,d,page,past,new,window,dtype", [
    (4, 2, 128, 64, [0, 40], [1, 1], 0, torch.float32),
    (12, 4, 64, 64, [300, 2], [1, 9], 0, torch.float32),
    (3, 1, 80, 64, [70], [5], 20, torch.float32),
    (8, 2, 32, 16, [33, 100], [1, 1], 0, torch.float32),
    (5, 5, 256, 64, [20], [3], 0, torch.float32),
    (4, 1, 96, 64, [64, 5], [2, 1], 0, torch.bfloat16),
    (2, 1, 128, 32, [64, 5], [1, 1], 12, torch.bfloat16),
    (1, 1, 16, 64, [600], [1], 0, torch.bfloat16),
])
def test_rows_in_32_bits(nq, nkv, d, page, past, new, window, dtype):
    st = Step(past, new, nkv, d, page, seed=nq + d)
    st.fill(d)
    check_attention(st, nq, dtype, window, nq)


@pytest.mark.parametrize("nkv,d,dtype", [(2, 128, torch.bfloat16), (1, 64, torch.bfloat16), (2, 128, torch.float32)])
@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("which", ["keys", "values"])
def test_a_token_that_is_not_finite_reaches_only_the_rows_that_see_it(nkv, d, dtype, window, which):
    st = Step([30, 90], [12, 1], nkv, d, seed=5)
    st.fill(5)
    slot, at = st.slots[0], 35
    part = getattr(st, which)
    part.scales[int(st.table[slot, at // 64]), :, at % 64] = 255
    seen = lambda s, p: s == slot and p >= at and (not window or p < at + window)
    check_attention(st, 4 * nkv, dtype, window, 2, expect_nan=seen)


def test_scores_that_spread_and_large_queries():
    st = Step([500, 0, 63], [1, 1, 1], 2, 128, seed=9)
    st.fill(9)
    check_attention(st, 4, torch.bfloat16, 0, 3, scale=1.0)              # weights from 1 to 2^-200
    check_attention(st, 4, torch.bfloat16, 0, 4, scale=0.0)              # all keys alike
    g = torch.Generator().manual_seed(1)
    q = torch.randn(3, 4 * 128, generator=g).bfloat16()
    outs = []
    for up in (1.0, 2.0 ** 60, 2.0 ** -60):
        out = torch.empty(3, 4 * 128, dtype=torch.bfloat16, device=DEV)
        ops.cache4_attention((q * up).to(DEV), 512, st.view(), st.batch(), out, 4, 2, 128, 0, 0.1 / up)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_queries_that_are_zero_or_not_finite():
    st = Step([70, 70, 70], [1, 1, 1], 1, 128, seed=9)
    st.fill(9)
    q = torch.randn(3, 2 * 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    q[0] = 0.0
    q[1, 3] = float("nan")
    out = torch.empty(3, 256, dtype=torch.bfloat16, device=DEV)
    ops.cache4_attention(q.to(DEV), 256, st.view(), st.batch(), out, 2, 1, 128, 0, 0.1)
    got = out.cpu()
    assert got[1, :128].isnan().all() and got[1, 128:].isfinite().all() and got[0].isfinite().all() and got[2].isfinite().all()
    v = plain.gathered(st.values, st.table, st.slots[0], 71, 64).mean(0)[0]
    assert ((got[0, :128].double() - v).abs() <= 2.0 ** -8 * v.abs() + 2.0 ** -10).all()


def test_offsets_beyond_32_bits():
    pages, nkv, d = 140000, 8, 128                   # 4.6 GB of codes each
    st = Step([130], [1], nkv, d, seed=2)
    st.fill(2)
    far = torch.tensor([pages - 1, 3, pages - 2], dtype=torch.int32)
    near = st.table[st.slots[0], :3].long()
    pool = lambda w: torch.full((pages, nkv, 64, w), 255, dtype=torch.uint8, device=DEV)
    parts = []
    for part in (st.keys, st.values):
        big = cb.Packed4(pool(d // 2), pool(d // 16))
        big.codes[far.long().to(DEV)] = part.codes[near].to(DEV)
        big.scales[far.long().to(DEV)] = part.scales[near].to(DEV)
        parts.append(big)
    table = st.table.clone()
    table[st.slots[0], :3] = far
    kv = cb.KVView(*parts, table.to(DEV), 64, cb.KVRequirement(nkv, d, packed4=True))
    q = torch.randn(1, 16 * d, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    a, b, c = (torch.empty(1, 16 * d, dtype=torch.bfloat16, device=DEV) for _ in range(3))
    ops.cache4_attention(q, 16 * d, st.view(), st.batch(), a, 16, nkv, d, 0, 0.1)
    ops.cache4_attention(q, 16 * d, kv, st.batch(), b, 16, nkv, d, 0, 0.1)
    assert torch.equal(a, b)
    w = torch.randn(1, 32 * d, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    s, p = on_device(torch.tensor(st.row_slot, dtype=torch.int32), torch.tensor(st.row_pos, dtype=torch.int32))
    small = st.view()
    for view in (small, kv):
        ops.cache4_append(w, view, s, p, 16, nkv, d, freqs(d).to(DEV), d, q_out=c)
    for x, y in zip(ops.cache4_read(small, s, p), ops.cache4_read(kv, s, p)):
        assert torch.equal(x, y)


def test_captured_steps_follow_the_lengths_and_share_nothing():
    """Two graphs of the same step replayed on two streams at once, with lengths that change between replays."""
    nq, nkv, d = 16, 4, 128
    lengths = [[100, 3, 1500], [1, 700, 64]]
    st = [Step([n - 1 for n in l], [1] * 3, nkv, d, seed=i, slots=4) for i, l in enumerate(lengths)]
    cases = []
    for i, s in enumerate(st):
        s.fill(i)
        q = torch.randn(3, nq * d, generator=torch.Generator().manual_seed(i)).bfloat16().to(DEV)
        view, batch = s.view(), s.batch()
        want = torch.empty(3, nq * d, dtype=torch.bfloat16, device=DEV)
        ops.cache4_attention(q, nq * d, view, batch, want, nq, nkv, d, 0, 0.1)
        short = torch.tensor([min(p, 40 + 9 * j) for j, p in enumerate(s.past)], dtype=torch.int32, device=DEV)
        want_short = torch.empty_like(want)
        batch_short = cb.StepBatch(batch.tokens, batch.row_slot, short, batch.seq_start, batch.seq_slot, short, batch.want_rows,
                                   slots=batch.slots, past=short.tolist(), n_new=[1] * 3)
        ops.cache4_attention(q, nq * d, view, batch_short, want_short, nq, nkv, d, 0, 0.1)
        out = torch.empty_like(want)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            ops.cache4_attention(q, nq * d, view, batch, out, nq, nkv, d, 0, 0.1)
        cases.append((graph, batch, out, want, short, want_short, view, q))
    streams = [torch.cuda.Stream() for _ in cases]
    longer = [c[1].row_pos.clone() for c in cases]
    for turn in range(6):
        for c, full in zip(cases, longer):
            c[1].row_pos.copy_(full if turn % 2 == 0 else c[4])
        torch.cuda.synchronize()
        for _ in range(5):
            for c, stream in zip(cases, streams):
                with torch.cuda.stream(stream):
                    c[0].replay()
        torch.cuda.synchronize()
        for c in cases:
            assert torch.equal(c[2], c[3] if turn % 2 == 0 else c[5])


def test_the_same_bits_every_time_and_on_another_stream():
    st = Step([4000, 17, 900, 2222], [1, 1, 1, 1], 2, 128, seed=4)
    st.fill(4)
    q = torch.randn(4, 8 * 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    view, batch = st.view(), st.batch()
    outs = []
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(6):
        out = torch.empty(4, 8 * 128, dtype=torch.bfloat16, device=DEV)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream if i % 2 else torch.cuda.default_stream()):
            ops.cache4_attention(q, 1024, view, batch, out, 8, 2, 128, 0, 0.1)
        torch.cuda.synchronize()
        outs.append(out)
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("lengths", [[900], [4000, 17, 900, 2222], [64] * 20])
def test_merging_by_the_last_block_or_by_a_second_kernel(monkeypatch, lengths):
    """Captured calls count in places of their own while there are any, and then do without: the same bits."""
    st = Step([n - 1 for n in lengths], [1] * len(lengths), 2, 128, seed=4)
    st.fill(4)
    q = torch.randn(len(lengths), 8 * 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    view, batch = st.view(), st.batch()
    outs, launches = [], []
    for spare in ("plain", "captured", "captured without"):
        if spare == "captured without":
            monkeypatch.setattr(ops, "_arrivals_spare", {})
        out = torch.empty(len(lengths), 8 * 128, dtype=torch.bfloat16, device=DEV)
        before = ops.launch_count()
        if spare == "plain":
            ops.cache4_attention(q, 1024, view, batch, out, 8, 2, 128, 0, 0.1)
        else:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                ops.cache4_attention(q, 1024, view, batch, out, 8, 2, 128, 0, 0.1)
            for _ in range(3):
                graph.replay()
        launches.append(ops.launch_count() - before)
        torch.cuda.synchronize()
        outs.append(out)
    assert launches == [1, 1, 2]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    assert all(int(c.abs().sum()) == 0 for c in ops._arrivals.values())


@pytest.mark.parametrize("nq,nkv,d,lengths", [(4, 1, 64, [9000, 40, 300]), (8, 1, 128, [20000]), (32, 1, 128, [9999, 700]), (8, 1, 256, [10000]),
                                                (4, 2, 128, [8090]), (3, 3, 128, [8090]), (2, 2, 128, [8100, 8090])])
def test_a_segment_of_many_blocks(monkeypatch, nq, nkv, d, lengths):
    """More parts than are merged at once: 32 neighbours first, then what they made; or by the second kernel in pieces of 32.  The order of
    additions differs between the two, so they may be a step of bfloat16 apart.  (8,090 keys are 253 units: 33 blocks, and the next
    segment begins in the last of them.)"""
    st = Step([n - 1 for n in lengths], [1] * len(lengths), nkv, d, seed=4)
    st.fill(4)
    got = check_attention(st, nq, torch.bfloat16, 0, 9)
    q = (1.5 * torch.randn(len(lengths), (nq + 2 * nkv) * d, generator=torch.Generator().manual_seed(9))).bfloat16().to(DEV)         # the same
    view, batch, outs = st.view(), st.batch(), []
    monkeypatch.setattr(ops, "_arrivals_spare", {})
    for _ in range(2):
        out = torch.empty(len(lengths), nq * d, dtype=torch.bfloat16, device=DEV)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        before = ops.launch_count()
        with torch.cuda.graph(graph):
            ops.cache4_attention(q, (nq + 2 * nkv) * d, view, batch, out, nq, nkv, d, 0, 1.0 / math.sqrt(d))
        assert ops.launch_count() - before == 2
        graph.replay()
        torch.cuda.synchronize()
        outs.append(out.cpu().double())
    assert torch.equal(outs[0], outs[1])
    assert ((outs[0] - got).abs() <= 2.0 ** -7 * got.abs() + 2.0 ** -15 * got.abs().max()).all()
    assert all(int(c.abs().sum()) == 0 for c in ops._arrivals.values())


def test_a_captured_step_of_runs_follows_the_device():
    """A captured step of two runs, replayed with the same rows dealt out otherwise: by the lengths on the device."""
    q = torch.randn(8, 4 * 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    outs = []
    for new in ([3, 5], [7, 1]):
        st = Step([100, 40], new, 1, 128, seed=6, slots=4)
        st.fill(6)
        batch, out = st.batch(), torch.empty(8, 256, dtype=torch.bfloat16, device=DEV)
        batch.runs4[2, 1, 128, 0, 512] = ("codes",)
        ops.cache4_attention(q, 512, st.view(), batch, out, 2, 1, 128, 0, 0.1)
        outs.append((st, st.batch(), out))
    (st, batch, want), (other, other_batch, other_want) = outs
    view, out = st.view(), torch.empty(8, 256, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache4_attention(q, 512, view, batch, out, 2, 1, 128, 0, 0.1)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    for name in ("row_slot", "row_pos", "seq_start", "seq_slot", "seq_past"):
        getattr(batch, name).copy_(getattr(other_batch, name))
    for mine, its in ((view.keys, other.view().keys), (view.values, other.view().values)):
        mine.codes.copy_(its.codes)
        mine.scales.copy_(its.scales)
    view.page_table.copy_(other.view().page_table)
    graph.replay()
    torch.cuda.synchronize()
    # (other tiles: either is off by half a step of bfloat16 and by 2^-11 of the weighted values, at most the largest)
    most = plain.values(other.values.codes, other.values.scales).nan_to_num(0.0).abs().max()
    got, wanted = out.cpu().double(), other_want.cpu().double()
    assert ((got - wanted).abs() <= 2.0 ** -7 * wanted.abs() + 2.0 ** -10 * most).all()


def test_refusals():
    st = Step([10], [2], 2, 64)
    kv, batch = st.view(), st.batch()
    q = torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device=DEV)
    out = torch.zeros(2, 4 * 64, dtype=torch.bfloat16, device=DEV)
    f = freqs(64).to(DEV)
    with pytest.raises(cb.CitlaliError, match="4 bits"):
        plain_kv = cb.KVView(out, out, kv.page_table, 64, cb.KVRequirement(2, 64))
        ops.cache4_attention(q, 512, plain_kv, batch, out, 4, 2, 64, 0, 0.1)
    with pytest.raises(cb.CitlaliError, match="pools"):
        ops.cache4_attention(q, 512, kv, batch, out, 4, 4, 64, 0, 0.1)
    with pytest.raises(cb.CitlaliError, match="queries"):
        ops.cache4_attention(q, 512, kv, batch, out.float(), 4, 2, 64, 0, 0.1)
    with pytest.raises(cb.CitlaliError, match="heads"):
        ops.cache4_attention(q, 512, kv, batch, torch.zeros(2, 3 * 64, dtype=torch.bfloat16, device=DEV), 3, 2, 64, 0, 0.1)
    with pytest.raises(cb.CitlaliError, match="rows do not fit"):
        ops.cache4_attention(q, 100, kv, batch, out, 4, 2, 64, 0, 0.1)
    with pytest.raises(cb.CitlaliError, match="window"):
        ops.cache4_attention(q, 512, kv, batch, out, 4, 2, 64, -3, 0.1)
    with pytest.raises(cb.CitlaliError, match="width"):
        ops.cache4_append(q, kv, batch.row_slot, batch.row_pos, 5, 2, 64, f, 64)
    with pytest.raises(cb.CitlaliError, match="rotated"):
        ops.cache4_append(q, kv, batch.row_slot, batch.row_pos, 4, 2, 64, f, 66)
    with pytest.raises(cb.CitlaliError, match="one a row"):
        ops.cache4_append(q, kv, batch.row_slot[:1], batch.row_pos, 4, 2, 64, f, 64)
    with pytest.raises(cb.CitlaliError, match="q_out"):
        ops.cache4_append(q, kv, batch.row_slot, batch.row_pos, 4, 2, 64, f, 64, q_out=out[:1])
    for over in (q[:, 64:320], torch.as_strided(q, (2, 256), (640, 1)), torch.as_strided(q, (2, 256), (256, 1))):
        with pytest.raises(cb.CitlaliError, match="not over their queries"):
            ops.cache4_append(q, kv, batch.row_slot, batch.row_pos, 4, 2, 64, f, 64, q_out=over)
    runs = Step([10], [2], 2, 64).batch()
    for way, words in ((("tiles", 0, 2, 3), "clusters"), (("tiles", 0, 2, 16), "clusters"), (("tiles", 0, 2, 0), "clusters")):
        runs.runs4[4, 2, 64, 0, 512] = way
        with pytest.raises(cb.CitlaliError, match=words):
            ops.cache4_attention(q, 512, kv, runs, out, 4, 2, 64, 0, 0.1)
    with pytest.raises(cb.CitlaliError, match="a row for every sequence"):
        many = Step([10, 3, 4], [1, 1, 1], 2, 64).batch()
        many.row_slot, many.row_pos = batch.row_slot, batch.row_pos
        ops.cache4_attention(q, 512, kv, many, out, 4, 2, 64, 0, 0.1)
    with pytest.raises(cb.CitlaliError, match="contiguous"):
        ops.cache4_append(q[:, ::2], kv, batch.row_slot, batch.row_pos, 2, 1, 64, f, 64)
    with pytest.raises(cb.CitlaliError, match="bfloat16 or float32"):
        ops.cache4_read(kv, batch.row_slot, batch.row_pos, dtype=torch.float16)
    with pytest.raises(cb.CitlaliError, match="float32 or bfloat16"):
        ops.cache4_append(q.half(), kv, batch.row_slot, batch.row_pos, 4, 2, 64, f, 64)


LONG_RUNS = [
    # nq, nkv, d, past, new, window
    (16, 8, 128, [0], [300], 0),
    (4, 2, 128, [65, 0, 500], [50, 130, 1], 0),
    (5, 1, 128, [200, 10], [64, 47], 100),
    (8, 2, 64, [0, 31], [129, 60], 0),
    (2, 1, 96, [0, 70], [70, 41], 33),
    (2, 2, 256, [3], [90], 0),
]


def check_long_run(st, nq, window, seed, expect_nan=None):
    """As check_attention, with the weights rounded to bfloat16 by the kernels for runs: half a step is 2^-8 of a weight."""
    g = torch.Generator().manual_seed(seed)
    nkv, d = st.nkv, st.d
    rows, pitch, scale = len(st.row_slot), (nq + 2 * nkv) * d, 1.0 / math.sqrt(d)
    q = (1.5 * torch.randn(rows, pitch, generator=g)).bfloat16()
    out = torch.full((rows + 1, nq * d), 5.0, dtype=torch.bfloat16, device=DEV)
    before = ops.launch_count()
    batch = st.batch()
    batch.runs4[nq, nkv, d, window, pitch] = ("pages",)      # whatever the times say
    ops.cache4_attention(q.to(DEV), pitch, st.view(), batch, out, nq, nkv, d, window, scale)
    got = out.cpu().double()
    assert (got[rows:] == 5.0).all()
    row = 0
    for s, past, n in zip(st.slots, st.past, st.new):
        k, v = (plain.gathered(part, st.table, s, past + n, st.page) for part in (st.keys, st.values))
        for i in range(n):
            o, weight, reach = plain.attention(q[row, :nq * d].view(nq, d), k, v, past + i, window, scale, nq // nkv)
            off = 4 * (d / 8 + 8) * 2.0 ** -23 * reach[:, None] + 2.0 ** -8 + (past + n + 64) / 32 * 2.0 ** -23
            have = got[row].view(nq, d)
            if expect_nan is not None and expect_nan(s, past + i):
                assert have.isnan().all()
            else:
                assert ((have - o).abs() <= 2.0 ** -8 * o.abs() + off * weight).all(), (s, past + i)
            row += 1
    return ops.launch_count() - before


@pytest.mark.parametrize("nq,nkv,d,past,new,window", LONG_RUNS)
def test_longer_runs(nq, nkv, d, past, new, window):
    st = Step(past, new, nkv, d, seed=nq + d)
    st.fill(sum(new))
    check_long_run(st, nq, window, nq)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", ["keys", "values"])
@pytest.mark.parametrize("window", [0, 20])
def test_a_token_that_is_not_finite_in_a_longer_run(d, which, window):
    st = Step([30, 10], [90, 50], 1, d, seed=5)
    st.fill(5)
    slot, at = st.slots[0], 75
    part = getattr(st, which)
    part.scales[int(st.table[slot, at // 64]), :, at % 64] = 255
    check_long_run(st, 2, window, 2, expect_nan=lambda s, p: s == slot and p >= at and (not window or p < at + window))


@pytest.mark.parametrize("way", [("codes",), ("pages",), ("tiles", 0, 4, 2)])
def test_queries_that_end_with_their_last_row(way):
    """Rows of a wider projection, and nothing behind the last row's queries."""
    st = Step([40, 0], [60, 30], 2, 128, seed=8)
    st.fill(8)
    rows, wide, pitch = 90, 4 * 128, 8 * 128
    q = torch.randn(rows, pitch, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    made = []
    for given in (q, q.flatten()[:(rows - 1) * pitch + wide].clone()):
        batch, out = st.batch(), torch.full((rows, wide), 5.0, dtype=torch.bfloat16, device=DEV)
        batch.runs4[4, 2, 128, 0, pitch] = way
        flag = torch.zeros(4, dtype=torch.int32, device=DEV)
        ops.cache4_attention(given, pitch, st.view(), batch, out, 4, 2, 128, 0, 0.1, error_flag=flag)
        made.append(out)
        assert not flag.any()                            # (no wait ran out)
    assert torch.equal(made[0], made[1])


def test_queries_over_the_rows_themselves():
    st = Step([5, 0], [1, 1], 2, 64, seed=3)
    s, p = on_device(torch.tensor(st.row_slot, dtype=torch.int32), torch.tensor(st.row_pos, dtype=torch.int32))
    made = []
    for how in (lambda x: None, lambda x: x[:, :256], lambda x: torch.empty(2, 256, dtype=x.dtype, device=DEV)):
        qkv, view = torch.randn(2, 512, generator=torch.Generator().manual_seed(4)).bfloat16().to(DEV), st.view()
        q_out = how(qkv)
        ops.cache4_append(qkv, view, s, p, 4, 2, 64, freqs(64).to(DEV), 64, q_out=q_out)
        made.append((qkv[:, :256] if q_out is None else q_out, view.keys.codes, view.values.codes))
    for other in made[1:]:
        assert all(torch.equal(a, b) for a, b in zip(made[0], other))


def test_longer_runs_a_few_sequences_at_a_time(monkeypatch):
    st = Step([0, 100, 5], [70, 60, 45], 2, 128, seed=8)
    st.fill(8)
    assert check_long_run(st, 4, 0, 1) == 2                              # one expansion, one attention
    monkeypatch.setattr(ops, "_EXPAND_BYTES", 1)
    assert check_long_run(st, 4, 0, 1) == 6
