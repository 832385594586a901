"""The paged 4-bit cache: block tables against a list of free blocks kept in Python, stored rows against the quantiser's definition,
attention against a softmax in 64 bits over what the codes stand for, and the three together as a step uses them."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(n_blocks=64, block=16, seqs=8, max_blocks=None, heads=16, kv=8, dim=64, layers=1):
    from vui_b200 import Kv4Cache

    return Kv4Cache(n_layers=layers, n_heads=heads, n_kv_heads=kv, head_dim=dim, n_blocks=n_blocks, block_size=block, max_seqs=seqs,
                    max_blocks=max_blocks)


# ----------------------------------------------------------------------------------------------------------- tables
class Tables:
    """What vuib_kv4_plan is documented to do, entry by entry."""

    def __init__(self, n_blocks, block, seqs, max_blocks):
        self.bs, self.max_blocks = block, max_blocks
        self.free = list(range(n_blocks))
        self.len = [0] * seqs
        self.table = [[-1] * max_blocks for _ in range(seqs)]

    def plan(self, slots, new, at, n_rows, max_new):
        seen, picked, bad = set(), [], False
        for i, s in enumerate(slots):
            if s == -1:
                continue
            if not 0 <= s < len(self.len) or s in seen:
                bad = True
                continue
            seen.add(s)
            start = self.len[s] if at is None else at[i]
            if not 0 <= start <= self.len[s] or not 0 <= new[i] <= max_new or start + new[i] > self.max_blocks * self.bs:
                bad = True
                continue
            picked.append((i, s, start, new[i]))
        rows, fit = 0, []
        for e in picked:
            rows += e[3]
            if rows <= n_rows:
                fit.append(e)
            else:
                bad = True
        up = lambda n: -(-n // self.bs)  # noqa: E731
        back = []
        for _, s, start, m in fit:
            for j in range(up(start + m), up(self.len[s])):
                back.append(self.table[s][j])
                self.table[s][j] = -1
        self.free += back[::-1]
        asked, have, out = 0, len(self.free), {}
        for i, s, start, m in fit:
            grow = max(0, up(start + m) - up(self.len[s]))
            asked += grow
            if grow and asked > have:
                bad = True
                continue
            for j in range(up(self.len[s]), up(start + m)):
                self.table[s][j] = self.free.pop()
            self.len[s] = start + m
            out[i] = [(s, p, self.table[s][p // self.bs] * self.bs + p % self.bs) for p in range(start, start + m)]
        cu, flat = [0], []
        for i in range(len(slots)):
            flat += out.get(i, [])
            cu.append(len(flat))
        flat += [(-1, -1, -1)] * (n_rows - len(flat))
        return cu, flat, bad


def check_tables(cache, plan, ref, want):
    from vui_b200._lib import VuibError

    cu, flat, bad = want
    assert plan.cu_rows.tolist() == cu
    got = list(zip(plan.row_slot.tolist(), plan.row_pos.tolist(), plan.slot_map.tolist()))
    assert got == flat
    assert cache.seq_lens.tolist() == ref.len
    assert cache.block_table.tolist() == ref.table
    n = int(cache.n_free.item())
    assert n == len(ref.free) and cache._free[:n].tolist() == ref.free
    if bad:
        with pytest.raises(VuibError):
            cache.check_device()
    cache.check_device()


@pytest.mark.parametrize("block, seqs, n_blocks, max_blocks, seed", [(16, 5, 12, 4, 0), (32, 40, 90, 6, 1), (64, 300, 500, 7, 2), (16, 1500, 4000, 9, 3), (256, 3, 5, 3, 4)])
def test_tables_over_many_steps(block, seqs, n_blocks, max_blocks, seed):
    """Growth, cut-backs, releases, sequences left out, entries that are out of range or named twice, too few rows, too few blocks."""
    r = random.Random(seed)
    cache, ref = make(n_blocks, block, seqs, max_blocks), Tables(n_blocks, block, seqs, max_blocks)
    for step in range(25):
        slots = r.sample(range(seqs), r.randint(1, seqs))
        kind = step % 5
        if kind == 3:
            slots = [r.choice((s, s, s, -1, slots[0], seqs, -7)) for s in slots]
        longest = max_blocks * block
        new = [r.choice((0, 1, 1, r.randint(0, longest // 2), longest + 1 if kind == 3 else 2)) for _ in slots]
        at = None
        if kind in (2, 4):
            at = [r.randint(0, ref.len[s]) if 0 <= s < seqs else 0 for s in slots]
            if kind == 4 and r.random() < 0.5:
                at, new = [0] * len(slots), [0] * len(slots)
        n_rows, max_new = sum(new), max(new)
        if kind == 1:
            n_rows, max_new = n_rows * 2 // 3, min(max_new, n_rows * 2 // 3)
        want = ref.plan(slots, new, at, n_rows, max_new)
        dev = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        plan = cache.plan(dev(slots), dev(new), at=dev(at), n_rows=n_rows, max_new=max_new) if step % 2 else \
            cache.plan(slots, new, at=at, n_rows=n_rows, max_new=max_new)
        check_tables(cache, plan, ref, want)


def test_one_row_each_and_release():
    cache, ref = make(40, 16, 6, 5), Tables(40, 16, 6, 5)
    for _ in range(35):
        want = ref.plan([3, 0, 5], [1, 1, 1], None, 3, 1)
        check_tables(cache, cache.plan([3, 0, 5]), ref, want)
    cache.release([0])
    ref.plan([0], [0], [0], 0, 0)
    assert cache.seq_lens.tolist() == ref.len and cache.block_table.tolist() == ref.table
    want = ref.plan([1], [70], None, 70, 70)
    check_tables(cache, cache.plan([1], [70]), ref, want)
    cache.reset()
    assert cache.seq_lens.tolist() == [0] * 6 and int(cache.n_free.item()) == 40 and (cache.block_table == -1).all()


# ------------------------------------------------------------------------------------------------------ stored rows
def stored(x):
    """The values that the codes of x (..., dim) stand for, by the definition (its steps are fp32): fp64."""
    g = x.float().unflatten(-1, (-1, 32))
    g = torch.where(g.isnan(), 0.0, g).clamp(-60000, 60000)
    zero = g.amin(-1, keepdim=True).half().float()
    scale = ((g.amax(-1, keepdim=True) - zero) * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)).half().float()
    code = torch.where(scale > 0, ((g - zero) / torch.where(scale > 0, scale, 1.0)).round().clamp(0, 15), 0.0)
    return (scale.double() * code.double() + zero.double()).half().double().flatten(-2)


def rows_of(kind, n, kv, dim, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, kv, dim, generator=g, device="cuda")
    if kind == "wide":
        x = x * torch.exp2(torch.randint(-20, 13, (n, kv, dim), generator=g, device="cuda").float())
    if kind == "flat":
        x = x[..., :1].expand(-1, -1, dim) * (torch.arange(dim, device="cuda") % 64 < 32)
    if kind == "small":
        x = x * 1e-6
    return x.bfloat16()


@pytest.mark.parametrize("dim, block, kv, kind", [(64, 16, 8, "normal"), (64, 256, 1, "wide"), (96, 32, 4, "flat"), (96, 64, 3, "small"),
                                                  (128, 128, 2, "wide"), (128, 16, 8, "flat")])
def test_stored_rows(dim, block, kv, kind):
    cache = make(60, block, 5, heads=kv, kv=kv, dim=dim)
    lens, seen = [0] * 5, {}
    for step, new in enumerate(([1, 0, 17, 5, 33], [15, 16, 1, 0, 2], [1, 1, 1, 1, 1])):
        plan = cache.plan([4, 1, 0, 3, 2], new)
        k, v = (rows_of(kind, sum(new), kv, dim, 10 * step + j) for j in (0, 1))
        cache.append(0, k, v, plan)
        for s, p, a, b in zip(plan.row_slot.tolist(), plan.row_pos.tolist(), stored(k), stored(v)):
            seen[s, p] = (a, b)
    places = sorted(seen, key=lambda x: (x[1] * 7919 + x[0]) % 97)
    got = cache.read(0, [s for s, _ in places], [p for _, p in places])
    cache.check_device()
    for j in (0, 1):
        want = torch.stack([seen[x][j] for x in places])
        assert torch.equal(got[j], want.bfloat16())       # f16 to bf16: one rounding of the same value
    # the code is the nearest of 16: half a step, the step's own rounding over 15 of them, and one to f16 of a value below 60000
    x = rows_of(kind, 50, kv, dim, 3)
    g = x.double().unflatten(-1, (-1, 32))
    span = (g.amax(-1) - g.amin(-1))[..., None]
    off = (stored(x).unflatten(-1, (-1, 32)) - g).abs()
    assert (off <= span / 30 * (1 + 2.0 ** -9) + span * 2.0 ** -11 + 3 * 2.0 ** -11 * g.abs().amax(-1, keepdim=True) + 2.0 ** -20).all()


def test_infinite_and_undefined_values_are_stored_as_finite_ones():
    from vui_b200._lib import VuibError

    cache = make(8, 16, 2, heads=2, kv=2)
    plan = cache.plan([1], [3])
    k = torch.ones(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    v = k.clone()
    k[0, 0, 0], k[1, 1, 40], v[2, 0, 63], v[1, 0, 0] = float("nan"), float("inf"), float("-inf"), 1e30
    cache.append(0, k, v, plan)
    with pytest.raises(VuibError, match="beyond"):
        cache.check_device()
    cache.check_device()
    got = cache.read(0, [1, 1, 1, -1], [0, 1, 2, 5])
    for x, want in zip(got, (k, v)):
        assert torch.equal(x[:3], stored(want).bfloat16()) and x.isfinite().all() and (x[3] == 0).all()
    assert got[0][1, 1, 40] == 59904 and got[1][2, 0, 63] == -59904     # 60000 in bf16


def test_reading_what_is_not_there_is_flagged():
    from vui_b200._lib import VuibError

    cache = make(8, 16, 2)
    cache.plan([0], [20])
    for s, p in ((0, 40), (1, 0), (2, 0), (-2, 0), (0, -1), (0, 1 << 20)):
        k, v = cache.read(0, [s], [p])
        assert (k == 0).all() and (v == 0).all()
        with pytest.raises(VuibError):
            cache.check_device()


def test_rows_that_lie_anywhere():
    """Views of a fused projection's output, other orders and types, unaligned starts; outputs into a stretch of a larger tensor."""
    cache = make(20, 16, 2, heads=8, kv=4)
    fused = torch.randn(40, (8 + 4 + 4) * 64, device="cuda").bfloat16()
    k, v = fused[:, 512:768].unflatten(1, (4, 64)), fused[:, 768:]
    plan = cache.plan([0], [40])
    slots, pos = [0] * 40, list(range(40))
    cache.append(0, k, v, plan)
    want = cache.read(0, slots, pos)
    assert torch.equal(want[0], stored(k).bfloat16()) and torch.equal(want[1].flatten(1), stored(v.unflatten(1, (4, 64))).bfloat16().flatten(1))
    odd = torch.empty(40 * 256 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(40, 4, 64)
    odd.copy_(k)
    for a, b in ((odd, v.float()), (k.transpose(0, 1).contiguous().transpose(0, 1), v.flip(0).flip(0)), (k.cpu(), v.cpu())):
        cache.append(0, torch.zeros_like(k), torch.zeros_like(v), plan)
        cache.append(0, a, b, plan)
        assert all(torch.equal(x, y) for x, y in zip(cache.read(0, slots, pos), want))
    big = torch.full((2, 50, 6, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    cache.read(0, slots, pos, k_out=big[0, 5:45, 1:5], v_out=big[1, 10:, :4])
    assert torch.equal(big[0, 5:45, 1:5], want[0]) and torch.equal(big[1, 10:, :4], want[1])
    assert (big[0, :5] == 7).all() and (big[0, 45:] == 7).all() and (big[0, :, 0] == 7).all() and (big[1, :, 4:] == 7).all()
    with pytest.raises(ValueError):
        cache.read(0, slots, pos, k_out=big[0, 5:45, 1:5].float())
    with pytest.raises(ValueError):
        cache.read(0, slots, pos, k_out=odd)
    q = fused[:, :512]
    out = torch.full((40, 1024), 3.0, device="cuda", dtype=torch.bfloat16)
    a = cache.attention(0, q.unflatten(1, (8, 64)), plan)
    cache.attention(0, q, plan, out=out[:, 256:768])
    assert torch.equal(out[:, 256:768], a.flatten(1)) and (out[:, :256] == 3).all() and (out[:, 768:] == 3).all()


# -------------------------------------------------------------------------------------------------------- attention
def fixed(x, k, v, p, mag, scale):
    """What fixed-point queries and weights may add to an error: x (rows, heads, dim), k and v (n, heads, dim), p (heads, rows, n).

    Queries enter as whole numbers of 2^-13 of the power of two below their largest element: exact (8 digits) but for elements below
    2^-6 of it, each half a unit off at most.  Weights times value scales enter in units of 2^-16 of the largest scale R, half a unit off at
    most, against codes up to 15.  Both kinds of errors are independent of one another: six standard deviations (a unit's over the
    square root of 12)."""
    unit = torch.exp2(x.abs().amax(-1).clamp(min=1e-300).log2().floor())                # (rows, heads)
    small = (x.abs() < unit[..., None] / 64).double()
    score = torch.einsum("rhd,nhd->rhn", small, k * k).amax(-1).sqrt() * unit * scale * 2.0 ** -13 / 12 ** 0.5 * 6
    span = (v.unflatten(-1, (-1, 32)).amax(-1) - v.unflatten(-1, (-1, 32)).amin(-1)).amax() / 15 * 1.001
    sums = k.shape[0] ** 0.5 * span * 15 * 2.0 ** -16 / 12 ** 0.5 * 6 * p.amax(-1).T     # the largest weight is 1 of the sum
    return 2 * score[..., None] * mag + sums[..., None]


class Filled:
    """A cache with sequences of the given lengths, stored in rounds so that their blocks lie in turn, and its contents in fp64."""

    def __init__(self, lens, heads, kv, dim, block, seed=0, spare=3, key_scale=1.0, max_blocks=None, turn=300, n_blocks=None):
        n = len(lens)
        self.lens, self.heads, self.kv, self.dim = list(lens), heads, kv, dim
        most = -(-(max(lens) + spare) // block)
        self.cache = make(n_blocks or sum(-(-(x + spare) // block) for x in lens) + 2, block, n + 2, max_blocks or most, heads, kv, dim)
        self.slots = [(3 * i + 1) % n if n % 3 else i for i in range(n)]
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.k = [torch.zeros(0, kv, dim, device="cuda", dtype=torch.float64) for _ in lens]
        self.v = list(self.k)
        self.key_scale = key_scale
        done = [0] * n
        while any(d < x for d, x in zip(done, lens)):
            new = [min(turn, x - d) for d, x in zip(done, lens)]
            self.add(new)
            done = [d + m for d, m in zip(done, new)]

    def add(self, new):
        plan = self.cache.plan(self.slots, new)
        n = sum(new)
        k = (torch.randn(n, self.kv, self.dim, generator=self.g, device="cuda") * self.key_scale).bfloat16()
        v = torch.randn(n, self.kv, self.dim, generator=self.g, device="cuda").bfloat16()
        self.cache.append(0, k, v, plan)
        k, v, a = stored(k), stored(v), 0
        for i, m in enumerate(new):
            self.k[i], self.v[i] = torch.cat([self.k[i], k[a:a + m]]), torch.cat([self.v[i], v[a:a + m]])
            a += m
        return plan

    def want(self, q, new, scale=None):
        """Softmax attention in 64 bits, the same of the values' magnitudes, and what fixed() says."""
        outs, mags, more, a = [], [], [], 0
        scale = self.dim ** -0.5 if scale is None else scale
        for i, m in enumerate(new):
            n = self.k[i].shape[0]
            k, v = (x[i].repeat_interleave(self.heads // self.kv, 1) for x in (self.k, self.v))
            x = q[a:a + m].double()
            s = torch.einsum("rhd,nhd->hrn", x, k) * scale
            late = torch.arange(n, device="cuda")[None, :] > torch.arange(n - m, n, device="cuda")[:, None]
            p = s.masked_fill(late, float("-inf")).softmax(-1)
            outs.append(torch.einsum("hrn,nhd->rhd", p, v))
            mags.append(torch.einsum("hrn,nhd->rhd", p, v.abs()))
            more.append(fixed(x, k, v, p, mags[-1], scale) if m and n else torch.zeros_like(mags[-1]))
            a += m
        return torch.cat(outs), torch.cat(mags), torch.cat(more)


def close(out, want):
    # one rounding to bf16 (2^-8 of the value); the weights' rounding to f16, where they are (2^-11 each), and what fp32 scores below 64 in
    # magnitude are off (128 products and sums of 2^-24 each: 2^-24 * 128 * 64 = 2^-11 in the exponent), both of the magnitudes that are added
    # up; what fixed-point operands add
    ref, mag, more = want
    err = (out.double() - ref).abs()
    assert (err <= 2.0 ** -8 * ref.abs() + 2.0 ** -10 * mag + more + 1e-30).all(), (err / mag).max()


EDGES = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 192, 255, 256, 257, 320, 511, 512, 513, 777, 1024]


@pytest.mark.parametrize("heads, kv, dim, block", [(16, 8, 64, 64), (8, 8, 64, 16), (12, 4, 96, 16), (28, 4, 128, 32), (32, 4, 64, 256),
                                                   (26, 2, 128, 128), (16, 1, 96, 64), (5, 5, 128, 16)])
def test_single_tokens(heads, kv, dim, block):
    f = Filled([n - 1 for n in EDGES], heads, kv, dim, block)
    new = [1] * len(EDGES)
    plan = f.add(new)
    q = torch.randn(len(EDGES), heads, dim, device="cuda", generator=f.g).bfloat16()
    out = f.cache.attention(0, q, plan)
    assert torch.equal(out, f.cache.attention(0, q, plan))
    close(out, f.want(q, new))
    f.cache.check_device()


@pytest.mark.parametrize("heads, kv, dim, block, before, new", [
    (16, 8, 64, 64, [0, 5, 300, 250, 64, 900], [37, 1, 0, 20, 64, 3]),
    (16, 8, 64, 16, [0], [200]),
    (12, 4, 96, 32, [100, 0, 511], [3, 130, 2]),
    (32, 8, 128, 128, [1000, 0], [150, 257]),
    (16, 1, 64, 64, [10, 700], [9, 70]),
    (8, 8, 128, 16, [3, 0, 260], [2, 1, 5]),
    (4, 4, 64, 64, [2000], [2]),
    (2, 2, 96, 256, [0, 40, 1], [600, 500, 700]),
    (16, 8, 64, 64, [20] * 40, [0] * 13 + [64] * 20 + [33] * 7),
    # 4096 query heads of rows and more, and 128 of a kv head: whole and partial tiles of 128, groups that do not divide them, sequences
    # without rows, more tiles than SMs and fewer
    (16, 8, 64, 16, [0], [256]),
    (16, 8, 64, 64, [1000, 0, 3, 40], [64, 0, 200, 1]),
    (28, 4, 64, 32, [0, 129, 700], [101, 19, 55]),
    (24, 8, 96, 64, [0, 300], [171, 43]),
    (30, 2, 96, 128, [1500], [131]),
    (15, 5, 128, 16, [127, 1, 0], [129, 128, 127]),
    (64, 4, 128, 256, [0, 0, 2000], [1, 8, 64]),
    (16, 16, 64, 64, [100, 5], [1100, 7]),
    # contexts beyond eight pieces of 512, whose pieces are longer
    (16, 8, 64, 256, [4400, 6700], [20, 9]),
    (8, 8, 96, 64, [4200], [30]),
    (6, 2, 128, 64, [5000, 4097], [7, 40]),
    (4, 1, 64, 64, [4500], [90]),
    (32, 8, 128, 32, [0, 0, 0, 900], [380, 257, 128, 5]),
])
def test_chunks_of_prompts(heads, kv, dim, block, before, new):
    f = Filled([max(x, 1) for x in before], heads, kv, dim, block, spare=max(new))
    if 0 in before:     # from the very first position
        z = [i for i, x in enumerate(before) if x == 0]
        f.cache.release([f.slots[i] for i in z])
        for i in z:
            f.k[i], f.v[i] = f.k[i][:0], f.v[i][:0]
    plan = f.add(new)
    q = torch.randn(sum(new), heads, dim, device="cuda", generator=f.g).bfloat16()
    out = f.cache.attention(0, q, plan)
    assert torch.equal(out, f.cache.attention(0, q, plan))
    close(out, f.want(q, new))
    f.cache.check_device()


@pytest.mark.parametrize("seqs", [31, 32, 33, 39, 63, 65, 66, 85, 97, 129, 1025])
def test_any_number_of_sequences(seqs):
    """Work is shared out by searching the sequences 32 at a time: numbers that leave a group of one, of two, and of none."""
    for heads, kv, dim, new in ((2, 1, 64, 1), (8, 2, 64, 1), (12, 2, 96, 1), (9, 1, 128, 1), (8, 2, 64, 7), (4, 1, 128, 40))[:6 if seqs < 130 else 2]:
        f = Filled([1 + 37 * i % 90 for i in range(seqs)], heads, kv, dim, 16, spare=new)
        plan = f.add([new] * seqs)
        q = torch.randn(seqs * new, heads, dim, device="cuda", generator=f.g).bfloat16()
        out = torch.full_like(q, float("nan"))
        f.cache.attention(0, q, plan, out=out)
        close(out, f.want(q, [new] * seqs))
        f.cache.check_device()


@pytest.mark.parametrize("heads, kv, dim, seqs, new", [(40, 8, 96, 64, 68), (12, 4, 96, 8, 200), (12, 4, 64, 40, 90), (16, 4, 128, 30, 71)])
def test_many_tiles_that_end_inside_a_warp(heads, kv, dim, seqs, new):
    """Columns that end within 32 of one another, over and over, call after call: all bits the same, none of them anywhere else."""
    f = Filled([200 + 5 * i % 190 for i in range(seqs)], heads, kv, dim, 64, spare=new)
    plan = f.add([new] * seqs)
    q = torch.randn(seqs * new, heads, dim, device="cuda", generator=f.g).bfloat16()
    big = torch.full((seqs * new + 2, heads + 2, dim), 5.0, device="cuda", dtype=torch.bfloat16)
    out = big[1:-1, 1:-1]
    f.cache.attention(0, q, plan, out=out)
    close(out, f.want(q, [new] * seqs))
    first = big.clone()
    for _ in range(20):
        f.cache.attention(0, q, plan, out=out)
    assert torch.equal(big, first) and (big[0] == 5).all() and (big[-1] == 5).all() and (big[:, 0] == 5).all() and (big[:, -1] == 5).all()
    f.cache.check_device()


def test_long_contexts():
    for lens, heads, kv, dim, new in (([40000, 9000], 8, 2, 64, [1, 1]), ([20000, 3], 4, 1, 128, [1, 1]), ([30000], 2, 1, 64, [40])):
        f = Filled([n - m for n, m in zip(lens, new)], heads, kv, dim, 256, turn=8000, spare=max(new))
        plan = f.add(new)
        q = torch.randn(sum(new), heads, dim, device="cuda", generator=f.g).bfloat16()
        close(f.cache.attention(0, q, plan), f.want(q, new))
        f.cache.check_device()


@pytest.mark.parametrize("heads, new", [(8, [1, 1]), (64, [1, 1]), (8, [20, 3]), (64, [70, 64])])
def test_offsets_beyond_32_bits(heads, new):
    """A pool of 4.6 GB, whose blocks are taken from the far end: every form of attention, rows in and out."""
    f = Filled([700, 90], heads, 8, 128, 256, max_blocks=8, n_blocks=14000)
    plan = f.add(new)
    assert int(plan.slot_map.min()) * 8 * 128 // 32 * 40 > 2 ** 32
    q = torch.randn(sum(new), heads, 128, device="cuda", generator=f.g).bfloat16()
    close(f.cache.attention(0, q, plan), f.want(q, new))
    for i, slot in enumerate(f.slots):
        n = f.k[i].shape[0]
        k, v = f.cache.read(0, [slot] * n, list(range(n)))
        assert torch.equal(k, f.k[i].bfloat16()) and torch.equal(v, f.v[i].bfloat16())
    f.cache.check_device()


@pytest.mark.parametrize("size", [1e-30, 2.0 ** -12, 1.0, 300.0, 1e30])
def test_queries_of_any_size(size):
    """A scale that brings the scores back to where they belong."""
    f = Filled([70, 300], 16, 8, 64, 64)
    plan = f.add([1, 1])
    q = (torch.randn(2, 16, 64, device="cuda", generator=f.g) * size).bfloat16()
    scale = 0.125 / size
    close(f.cache.attention(0, q, plan, scale=scale), f.want(q, [1, 1], scale))


def test_peaked_scores():
    """Keys of 30: one position takes nearly all the weight, and the maximum moves from step to step.  Scores reach about 450, where 2^-24 *
    64 * 450 * log2(e) = 2^-10.6 in the exponent takes the place of the 2^-11 that close() allows for: twice that."""
    f = Filled([500, 40, 1500], 16, 8, 64, 64, key_scale=30.0)
    plan = f.add([1, 1, 1])
    q = torch.randn(3, 16, 64, device="cuda", generator=f.g).bfloat16()
    ref, mag, more = f.want(q, [1, 1, 1])
    close(f.cache.attention(0, q, plan), (ref, 2 * mag, more))


@pytest.mark.parametrize("heads, kv, dim, grow, new", [
    (16, 8, 64, False, 250), (8, 2, 128, True, 250), (6, 2, 96, True, 250), (16, 8, 64, True, 250),
    (16, 8, 64, False, 270), (16, 2, 64, True, 270), (32, 4, 128, True, 270), (24, 8, 96, True, 270), (32, 2, 128, False, 257)])
def test_peaked_chunks(heads, kv, dim, grow, new):
    """The same for chunks of prompts; with keys that grow along the sequence, so that a column's maximum keeps leaving the weights' range.
    Scores as above, of up to 450."""
    f = Filled([1], heads, kv, dim, 64, spare=1800, key_scale=30.0, max_blocks=40)
    for part in range(6):
        f.key_scale = 30.0 * (2.0 ** (part - 5) if grow else 1.0)
        plan = f.add([new])
        q = torch.randn(new, heads, dim, device="cuda", generator=f.g).bfloat16()
        ref, mag, more = f.want(q, [new])
        out = f.cache.attention(0, q, plan)
        close(out, (ref, 2 * mag, more))
        assert torch.equal(out, f.cache.attention(0, q, plan))
    f.cache.check_device()


@pytest.mark.parametrize("new, dim", [(100, 64), (300, 64), (300, 128)])
def test_a_row_of_nan_in_a_chunk(new, dim):
    f = Filled([700], 16, 8, dim, 64, spare=new)
    plan = f.add([new])
    q = torch.randn(new, 16, dim, device="cuda", generator=f.g).bfloat16()
    want = f.want(q, [new])
    bad = q.clone()
    bad[31, 7, 5], bad[90, 2, 0] = float("nan"), float("inf")
    out = f.cache.attention(0, bad, plan)
    assert out[31, 7].isnan().all() and out[90, 2].isnan().all()
    out[31, 7], out[90, 2] = want[0][31, 7].bfloat16(), want[0][90, 2].bfloat16()
    close(out, want)


def test_a_row_of_nan_stays_its_own():
    f = Filled([100, 400, 30], 16, 8, 64, 64)
    plan = f.add([2, 2, 2])
    q = torch.randn(6, 16, 64, device="cuda", generator=f.g).bfloat16()
    want = f.want(q, [2, 2, 2])
    bad = q.clone()
    bad[2, 3, 5] = float("nan")
    out = f.cache.attention(0, bad, plan)
    assert out[2, 3].isnan().all()
    out[2, 3] = want[0][2, 3].bfloat16()
    close(out, want)


def test_a_rows_bits_are_its_own():
    """Single tokens: whatever else is in the batch, however large the cache, wherever the blocks lie."""
    outs = []
    for others, block, mb in (([], 64, None), ([5, 1000, 77], 16, 100), ([300] * 60, 64, 200)):
        f = Filled([899] + others, 16, 8, 64, block, seed=5, turn=5000, max_blocks=mb)
        g = torch.Generator(device="cuda").manual_seed(77)
        k, v, q = (torch.randn(900, h, 64, generator=g, device="cuda").bfloat16() for h in (8, 8, 16))
        plan = f.cache.plan(f.slots[:1], [900], at=[0])
        f.cache.append(0, k, v, plan)
        f.cache.plan(f.slots[:1], [0], at=[899])
        plan = f.cache.plan(f.slots)
        rows = [k[-1:]] + [torch.zeros_like(k[:1])] * len(others), [v[-1:]] + [torch.zeros_like(v[:1])] * len(others)
        f.cache.append(0, torch.cat(rows[0]), torch.cat(rows[1]), plan)
        outs.append(f.cache.attention(0, q[:1].expand(1 + len(others), -1, -1).contiguous(), plan)[0])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_padding_rows_are_left_as_they_were():
    f = Filled([50, 20, 300], 16, 8, 64, 64)
    cache = f.cache
    before = cache._pool.clone()
    slots = torch.tensor([f.slots[0], -1, f.slots[2], -1], dtype=torch.int32, device="cuda")
    plan = cache.plan(slots, torch.tensor([1, 1, 3, 1], dtype=torch.int32, device="cuda"), n_rows=8, max_new=3)
    assert plan.cu_rows.tolist() == [0, 1, 1, 4, 4] and plan.row_slot.tolist()[4:] == [-1] * 4
    k, v = (torch.randn(8, 8, 64, device="cuda", generator=f.g).bfloat16() for _ in range(2))
    k[4:], v[4:] = float("nan"), float("inf")
    cache.append(0, k, v, plan)
    q = torch.randn(8, 16, 64, device="cuda", generator=f.g).bfloat16()
    q[4:] = float("nan")
    out = torch.full_like(q, 9.0)
    cache.attention(0, q, plan, out=out)
    cache.check_device()
    assert (out[4:] == 9).all()
    for i, a, b in ((0, 0, 1), (2, 1, 4)):
        f.k[i], f.v[i] = torch.cat([f.k[i], stored(k[a:b])]), torch.cat([f.v[i], stored(v[a:b])])
    close(out[:4], f.want(q[:4], [1, 0, 3]))
    # four rows of 8 kv heads, keys and values: 40 bytes each, and nothing else has changed
    assert int((cache._pool != before).sum()) <= 4 * 8 * 80


# --------------------------------------------------------------------------------------------------- as it is used
def test_captured_steps_cross_blocks():
    """Steps replayed from a graph, tables and all, are the same as eager ones; two caches' graphs replay side by side."""
    def fill():
        cache = make(60, 16, 3, 12, layers=2)
        g = torch.Generator(device="cuda").manual_seed(1)
        data = [torch.randn(45, 3, h, 64, generator=g, device="cuda").bfloat16() for h in (8, 8, 16)]
        return cache, data

    def step(cache, k, v, q):
        plan = cache.plan(slots, ones, n_rows=3, max_new=1)
        out = []
        for layer in range(2):
            cache.append(layer, k + layer, v, plan)
            out.append(cache.attention(layer, q, plan))
        return plan, out

    slots, ones = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([2, 0, 1], [1, 1, 1]))
    eager, data = fill()
    want = [step(eager, *(d[i] for d in data)) for i in range(45)]
    runs = []
    for _ in range(2):
        cache, _ = fill()
        bufs = [d[0].clone() for d in data]
        step(cache, *bufs)
        cache.reset()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan, out = step(cache, *bufs)
        cache.reset()
        runs.append((cache, bufs, graph, plan, out, torch.cuda.Stream()))
    for i in range(45):
        for cache, bufs, graph, plan, out, stream in runs:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                for b, d in zip(bufs, data):
                    b.copy_(d[i])
                graph.replay()
        torch.cuda.synchronize()
        for cache, bufs, graph, plan, out, stream in runs:
            assert torch.equal(plan.slot_map, want[i][0].slot_map) and torch.equal(plan.row_pos, want[i][0].row_pos)
            assert all(torch.equal(a, b) for a, b in zip(out, want[i][1]))
    for cache, *_ in runs:
        cache.check_device()
        assert cache.seq_lens.tolist() == [45] * 3


def test_captured_chunks():
    """Two caches' graphs of whole prompt chunks, replayed side by side for chunks of other lengths, are the same as eager calls."""
    def step(cache, bufs):
        k, v, q, new, at = bufs
        plan = cache.plan(slots, new, at=at, n_rows=320, max_new=300)
        cache.append(0, k, v, plan)
        return plan, cache.attention(0, q, plan, out=torch.full_like(q, 5.0))

    slots = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(9)
    runs = []
    for _ in range(2):
        cache, eager = make(120, 16, 3, 40), make(120, 16, 3, 40)
        bufs = [torch.randn(320, h, 64, generator=g, device="cuda").bfloat16() for h in (8, 8, 16)]
        bufs += [torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2)]
        step(cache, bufs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan, out = step(cache, bufs)
        runs.append((cache, eager, bufs, graph, plan, out, torch.cuda.Stream()))
    for new, at in (([300, 1, 19], [0, 0, 0]), ([0, 200, 120], [300, 1, 19]), ([20, 0, 300], [300, 0, 139]), ([0, 0, 0], [320, 0, 0]),
                    ([290, 30, 0], [320, 0, 0]), ([1, 1, 1], [610, 30, 0])):
        for cache, eager, bufs, graph, plan, out, stream in runs:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                for b in bufs[:3]:
                    b.normal_(generator=g)
                for b, x in zip(bufs[3:], (new, at)):
                    b.copy_(torch.tensor(x, dtype=torch.int32))
                graph.replay()
        torch.cuda.synchronize()
        for cache, eager, bufs, graph, plan, out, stream in runs:
            want_plan, want = step(eager, bufs)
            assert torch.equal(plan.slot_map, want_plan.slot_map) and torch.equal(out, want) and (out[sum(new):] == 5).all()
            cache.check_device()
            eager.check_device()


def test_one_plan_on_two_streams():
    """Two layers of one plan at the same time: each stream has partial sums of its own."""
    for new, heads, kv in (([1, 1], 16, 8), ([20, 40], 16, 8), ([300, 9], 16, 8)):
        f = Filled([3000, 800], heads, kv, 64, 64, spare=max(new))
        plan = f.add(new)
        qs = [torch.randn(sum(new), heads, 64, device="cuda", generator=f.g).bfloat16() for _ in range(2)]
        want = [f.cache.attention(0, q, plan) for q in qs]
        streams = [torch.cuda.Stream() for _ in qs]
        got = [[], []]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for _ in range(8):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i].append(f.cache.attention(0, qs[i], plan))
        torch.cuda.synchronize()
        assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


def test_on_another_stream():
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        f = Filled([200, 30], 16, 8, 64, 32)
        plan = f.add([1, 1])
        q = torch.randn(2, 16, 64, device="cuda", generator=f.g).bfloat16()
        out = f.cache.attention(0, q, plan)
    side.synchronize()
    close(out, f.want(q, [1, 1]))


def test_a_conversation_is_put_away_and_taken_up_again(nano_model):
    """An engine's bf16 rows into the 4-bit cache and back into another slot of the engine: attention over both is the same."""
    from vui_b200 import Engine

    eng = Engine(model=nano_model, max_rows=2, max_seq=512)
    row = eng.new_row()
    n = 201
    eng.prefill_ids(row, torch.randint(0, 151936, (n,), generator=torch.Generator().manual_seed(2)))
    layers = [0, 11, 23]
    cache = make(10, 64, 2, layers=len(layers))
    plan = cache.plan([1], [n])
    other = 1 - row.idx
    for i, layer in enumerate(layers):
        kv = eng.flash_kv_caches[layer]
        cache.append(i, kv.k_cache[row.idx, :n], kv.v_cache[row.idx, :n], plan)
        cache.read(i, plan.row_slot, plan.row_pos, k_out=kv.k_cache[other, :n], v_out=kv.v_cache[other, :n])
        k, v = stored(kv.k_cache[row.idx, :n]), stored(kv.v_cache[row.idx, :n])
        assert torch.equal(kv.k_cache[other, :n], k.bfloat16()) and torch.equal(kv.v_cache[other, :n], v.bfloat16())
        q = torch.randn(1, 1024, device="cuda", generator=torch.Generator(device="cuda").manual_seed(layer)).bfloat16()
        last = cache.plan([1], [1], at=[n - 1])
        cache.append(i, kv.k_cache[row.idx, n - 1:n], kv.v_cache[row.idx, n - 1:n], last)
        a = cache.attention(i, q, last).double()
        b = eng._attention(layer, q, torch.tensor([other]), torch.tensor([n - 1])).double()
        # both against the same in 64 bits: the bf16 slot holds keys and values rounded once more (2^-8 of each), which moves a score by at
        # most 2^-8 times the sum of its products' magnitudes
        kk, vv = (x.repeat_interleave(2, 1) for x in (k, v))
        qh = q.double().view(16, 64)
        p = (torch.einsum("hd,nhd->hn", qh, kk) / 8).softmax(-1)
        ref = torch.einsum("hn,nhd->hd", p, vv).flatten()
        mag = torch.einsum("hn,nhd->hd", p, vv.abs()).flatten()
        move = torch.einsum("hd,nhd->hn", qh.abs(), kk.abs()).amax(-1).repeat_interleave(64) / 8 * 2.0 ** -8
        more = fixed(qh[None], kk, vv, p[:, None], mag.view(1, 16, 64), 0.125).flatten()
        assert ((a[0] - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -10 * mag + more).all()
        assert ((b[0] - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.2 * move + 2.0 ** -10) * mag).all()
    cache.check_device()
    eng.check_device()


def test_refusals():
    from vui_b200._lib import VuibError

    cache = make(10, 16, 3, heads=16, kv=8)
    plan = cache.plan([0, 1], [2, 3])
    other = make(10, 16, 300, heads=16, kv=8).plan([280, 1], [2, 3])      # of another cache
    k, q = (torch.zeros(5, h, 64, device="cuda", dtype=torch.bfloat16) for h in (8, 16))
    for bad in (lambda: cache.append(0, k[:4], k[:4], plan), lambda: cache.append(0, q, q, plan), lambda: cache.attention(0, k, plan),
                lambda: cache.attention(0, q, plan, scale=0.0), lambda: cache.attention(0, q, plan, scale=-1.0),
                lambda: cache.attention(0, q, plan, scale=float("nan")), lambda: cache.attention(0, q, plan, out=q.float()),
                lambda: cache.attention(0, q, plan, out=q[:, :8]), lambda: cache.plan([]), lambda: cache.plan([0.5]), lambda: cache.plan([[0]]),
                lambda: cache.plan([0, 1], [1]), lambda: cache.plan([0], [1], at=[0, 0]), lambda: cache.read(0, [0, 1], [0]),
                lambda: cache.plan([0], torch.ones(1, dtype=torch.int32, device="cuda")), lambda: cache.plan([0], [1], n_rows=-1),
                lambda: cache.read(0, [0], [0], k_out=k[:1, :, :32]), lambda: cache.plan([2 ** 32]), lambda: cache.plan([0], [2 ** 40], n_rows=1),
                lambda: cache.attention(0, q, other), lambda: cache.append(0, k, k, other), lambda: cache.attention(0, q, None)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cache.append(1, k, k, plan), lambda: cache.attention(-1, q, plan), lambda: cache.read(7, [0], [0])):
        with pytest.raises(VuibError, match="layer"):
            bad()
    cache.check_device()
    assert cache.seq_lens.tolist() == [2, 3, 0]
    empty = cache.plan([0, 1], [0, 0])
    assert cache.attention(0, q[:0], empty).shape == (0, 16, 64)
    cache.append(0, k[:0], k[:0], empty)
    assert [x.shape for x in cache.read(0, [], [])] == [(0, 8, 64)] * 2
