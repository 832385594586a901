"""The paged 4-bit cache where it can go wrong: what blocks held before, outliers, sizes and values at the borders of what a call takes."""
import subprocess
import sys

import pytest
import torch
from test_gpu_kv4 import Filled, close, fixed, make, stored

pytestmark = pytest.mark.gpu


# columns of a tile (rows x query heads of a kv head): 1 to 4, at every width
FEW = [(8, 8, 64), (16, 8, 64), (9, 3, 64), (16, 4, 64), (4, 4, 96), (12, 4, 96), (2, 2, 128), (4, 2, 128), (32, 8, 128)]


@pytest.mark.parametrize("heads, kv, dim", FEW + [(16, 2, 64), (32, 2, 128)])
def test_what_a_block_held_before_does_not_count(heads, kv, dim):
    """Sequences that end inside a tile whose other positions still hold what was there before: another sequence's values, or the
    sequence's own from before a cut-back.  The same bits as in a cache where nothing was."""
    lens = [*range(1, 18), 33, 70, 650]
    g = torch.Generator(device="cuda").manual_seed(3)
    n = sum(lens)
    k, v, q = ((torch.randn(n, h, dim, generator=g, device="cuda") * s).bfloat16() for h, s in ((kv, 1), (kv, 0.5), (heads, 1)))
    q = q[:len(lens)].contiguous()
    last = torch.tensor(lens, device="cuda").cumsum(0) - 1
    before = torch.ones(n, dtype=torch.bool, device="cuda")
    before[last] = False
    outs = []
    for kind in ("fresh", "another's", "its own"):
        cache = make(sum(-(-x // 16) + 2 for x in lens), 16, len(lens), heads=heads, kv=kv, dim=dim)
        slots = list(range(len(lens)))
        if kind != "fresh":
            more = [x + 17 for x in lens]
            big = [((torch.rand(sum(more), kv, dim, generator=g, device="cuda") - 0.5) * 60000).bfloat16() for _ in range(2)]
            cache.append(0, *big, cache.plan(slots, more))
        plan = cache.plan(slots, [x - 1 for x in lens], at=[0] * len(lens) if kind == "its own" else None) if kind != "another's" else None
        if kind == "another's":
            cache.release(slots)
            plan = cache.plan(slots, [x - 1 for x in lens])
        cache.append(0, k[before], v[before], plan)
        plan = cache.plan(slots)
        cache.append(0, k[last], v[last], plan)
        outs.append(cache.attention(0, q, plan))
        cache.check_device()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("heads, kv, dim, new", [(8, 8, 64, 2), (8, 8, 64, 4), (16, 8, 64, 2), (4, 4, 96, 3), (4, 2, 96, 2), (2, 2, 128, 2), (8, 4, 128, 2)])
def test_later_rows_do_not_count(heads, kv, dim, new):
    """A chunk's first row has the same bits whatever the rows behind it store."""
    outs = []
    for size in (1.0, 20000.0):
        f = Filled([1, 21, 60, 700], heads, kv, dim, 64, spare=new)
        g = torch.Generator(device="cuda").manual_seed(4)
        k, v, q = (torch.randn(4 * new, h, dim, generator=g, device="cuda").bfloat16() for h in (kv, kv, heads))
        v.view(4, new, kv, dim)[:, 1:] *= size
        plan = f.cache.plan(f.slots, [new] * 4)
        f.cache.append(0, k, v, plan)
        outs.append(f.cache.attention(0, q, plan).view(4, new, heads, dim))
    assert torch.equal(outs[0][:, 0], outs[1][:, 0]) and not torch.equal(outs[0], outs[1])


def weighed(x, k, v, p, mag, scale):
    """As fixed(), with the weights' part taken from what is summed: weights times value scales enter in units of 2^-16 of the largest such
    product of a query and group of 32 elements, up to 1.01 of it, half a unit off each, against codes up to 15; independent errors, six
    standard deviations."""
    span = (v.unflatten(-1, (-1, 32)).amax(-1) - v.unflatten(-1, (-1, 32)).amin(-1)) / 15 * 1.001      # (n, heads, groups)
    unit = 1.01 * torch.einsum("hrn,nhg->rhgn", p, span).amax(-1) * 2.0 ** -16
    sums = k.shape[0] ** 0.5 * 15 * 6 / 12 ** 0.5 * unit.repeat_interleave(32, -1)
    return fixed(x, k, torch.zeros_like(v), p, mag, scale) + sums


@pytest.mark.parametrize("heads, kv, dim", FEW)
@pytest.mark.parametrize("size", [1000.0, 30000.0])
def test_outliers_of_no_weight(heads, kv, dim, size):
    """Positions with values far larger than the others' and next to no weight: the others lose nothing by them."""
    f = Filled([1], heads, kv, dim, 64, spare=1200, max_blocks=20)
    for n in (40, 300, 900):
        plan = f.cache.plan(f.slots, [n], at=[0])
        k, v = (torch.randn(n, kv, dim, generator=f.g, device="cuda") for _ in range(2))
        k[3::50], v[3::50] = -30.0, v[3::50] * size
        k, v = k.bfloat16(), v.clamp(-60000, 60000).bfloat16()
        f.cache.append(0, k, v, plan)
        f.k[0], f.v[0] = stored(k), stored(v)
        plan = f.cache.plan(f.slots, [1], at=[n - 1])
        f.cache.append(0, k[-1:], v[-1:], plan)
        q = torch.randn(1, heads, dim, device="cuda", generator=f.g).abs().bfloat16()
        ref, mag, _ = f.want(q, [1])
        kk, vv = (x[0].repeat_interleave(heads // kv, 1) for x in (f.k, f.v))
        p = (torch.einsum("rhd,nhd->hrn", q.double(), kk) * dim ** -0.5).softmax(-1)
        close(f.cache.attention(0, q, plan), (ref, mag, weighed(q.double(), kk, vv, p, mag, dim ** -0.5)))


def test_plans_at_the_border_of_a_blocks_shared_memory():
    """Numbers of sequences whose tables take about as much shared memory as a launch gets unasked, as a process's first plans."""
    program = """
from vui_b200 import Kv4Cache
for seqs, slots in ((1000, 4096), (1023, 4096), (1340, 1500), (1365, 1365), (1022, 4096), (4096, 4096)):
    cache = Kv4Cache(n_layers=1, n_heads=2, n_kv_heads=1, head_dim=64, n_blocks=seqs + 1, block_size=16, max_seqs=slots, max_blocks=2)
    plan = cache.plan(list(range(seqs)))
    cache.check_device()
    assert plan.cu_rows.tolist() == list(range(seqs + 1)) and cache.seq_lens.tolist() == [1] * seqs + [0] * (slots - seqs)
print("fine")
"""
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]


def test_positions_behind_a_sequences_end_are_not_read():
    """In a block that holds what another sequence left there."""
    from vui_b200._lib import VuibError

    cache = make(2, 32, 2, heads=2, kv=2)
    x = torch.full((64, 2, 64), 77.0, device="cuda", dtype=torch.bfloat16)
    cache.append(0, x, x, cache.plan([1], [64]))
    cache.release([1])
    plan = cache.plan([0], [20])
    cache.append(0, x[:20] * 0 + 5, x[:20] * 0 + 5, plan)
    for t in cache.read(0, [0] * 20, list(range(20))):
        assert (t == 5).all()
    cache.check_device()
    for p in (20, 21, 31, 32):
        for t in cache.read(0, [0, 0], [p, 19]):
            assert (t[0] == 0).all() and (t[1] == 5).all()
        with pytest.raises(VuibError, match="position"):
            cache.check_device()
    cache.plan([0], [0], at=[3])
    assert all((t == 0).all() for t in cache.read(0, [0], [3]))
    with pytest.raises(VuibError, match="position"):
        cache.check_device()
    assert all((t == 5).all() for t in cache.read(0, [0], [2]))
    cache.check_device()


def test_numbers_beyond_32_bits_on_the_device():
    """They are as out of range as any other, not what is left of them in 32 bits."""
    from vui_b200._lib import VuibError

    far = lambda *v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
    cache = make(10, 16, 3)
    cache.plan([0, 1], [5, 5])
    for call in (lambda: cache.plan(far(2 ** 32)), lambda: cache.plan(far(-2 ** 32)), lambda: cache.plan(far(2 ** 32 - 1)),
                 lambda: cache.plan(far(0), far(2 ** 32 + 1), n_rows=4, max_new=4),
                 lambda: cache.plan(far(0), far(1), at=far(2 ** 33 + 2), n_rows=4, max_new=4), lambda: cache.release(far(2 ** 32 + 1)),
                 lambda: cache.read(0, far(2 ** 32), far(0)), lambda: cache.read(0, far(0), far(2 ** 32 + 1))):
        call()
        with pytest.raises(VuibError):
            cache.check_device()
        assert cache.seq_lens.tolist() == [5, 5, 0]
    plan = cache.plan(far(1, -1), far(2, 0), at=far(4, 0), n_rows=4, max_new=4)
    assert plan.row_pos.tolist() == [4, 5, -1, -1] and cache.seq_lens.tolist() == [5, 6, 0]
    cache.check_device()


def test_unsigned_numbers():
    from vui_b200._lib import VuibError

    cache = make(10, 16, 3)
    for where in ("cpu", "cuda"):
        for t in (torch.uint8, torch.uint16, torch.uint32):
            assert cache.plan(torch.tensor([1]).to(t).to(where)).row_slot.tolist() == [1]
        with pytest.raises(ValueError):
            cache.plan(torch.tensor([1]).to(torch.uint64).to(where))
    far = torch.tensor([2 ** 32 - 1], dtype=torch.uint32)
    with pytest.raises(ValueError, match="32 bits"):
        cache.plan(far)
    cache.check_device()
    assert cache.plan(far.cuda()).row_slot.tolist() == [-1]
    with pytest.raises(VuibError):
        cache.check_device()


def test_sizes_beyond_32_bits():
    from vui_b200._lib import VuibError

    cache = make(10, 16, 3)
    plan = cache.plan([0], [1])
    k, q = (torch.zeros(1, h, 64, device="cuda", dtype=torch.bfloat16) for h in (8, 16))
    for bad in (lambda: cache.append(2 ** 32, k, k, plan), lambda: cache.attention(2 ** 32, q, plan), lambda: cache.read(-2 ** 32, [0], [0])):
        with pytest.raises(VuibError, match="layer"):
            bad()
    for n in (2 ** 24 + 1, 2 ** 31, 2 ** 32 + 1):
        with pytest.raises(ValueError, match="n_rows"):
            cache.plan([0], [1], n_rows=n, max_new=1)
    with pytest.raises(ValueError, match="n_rows"):
        cache.plan([0, 1], [2 ** 31 - 1, 2 ** 31 - 1])
    cache.check_device()
    assert cache.seq_lens.tolist() == [1, 0, 0]


def test_scales_that_are_0_in_32_bits():
    f = Filled([70], 16, 8, 64, 64)
    plan = f.add([1])
    q = torch.randn(1, 16, 64, device="cuda", generator=f.g).bfloat16()
    for scale in (1e-50, 1e-46, 5e-324, 1e31, float("inf")):
        with pytest.raises(ValueError, match="scale"):
            f.cache.attention(0, q, plan, scale=scale)
    for scale in (1e-40, 2.0 ** -126):
        close(f.cache.attention(0, q, plan, scale=scale), f.want(q, [1], scale))


@pytest.mark.parametrize("seqs, first", [(600, 100), (4096, 100), (600, 0)])
def test_lengths_whose_sum_is_beyond_32_bits(seqs, first):
    """Each in range by itself; all but the first are left as they are."""
    from vui_b200._lib import VuibError

    most = 1 << 22
    cache = make(64, 256, seqs, most // 256, heads=2, kv=1)
    new = torch.full((seqs,), most, dtype=torch.int32, device="cuda")
    new[0] = first
    for at in (None, torch.zeros_like(new)):
        plan = cache.plan(list(range(seqs)), new, at=at, n_rows=most, max_new=most)
        with pytest.raises(VuibError, match="more rows" if first else "more rows.*out of blocks"):
            cache.check_device()
        assert cache.seq_lens.tolist() == [first] + [0] * (seqs - 1) and int(cache.n_free.item()) == 64 - (first > 0)
        assert plan.cu_rows.tolist() == [0] + [first] * seqs and (plan.row_slot[first:] == -1).all() and (plan.slot_map[first:] == -1).all()
        assert plan.row_pos[:first].tolist() == list(range(first)) and int((cache.block_table >= 0).sum()) == (first > 0)
        cache.release([0])
        cache.check_device()
    plan = cache.plan([0, 5], [20, 1])
    assert plan.cu_rows.tolist() == [0, 20, 21]
    cache.check_device()


FORMS = [(16, 8, 64, 1), (16, 4, 64, 1), (12, 4, 96, 1), (4, 2, 128, 1), (32, 8, 128, 1), (16, 2, 64, 1), (26, 2, 128, 1), (12, 2, 96, 3), (4, 4, 64, 20),
         (16, 8, 64, 150), (12, 4, 96, 180), (32, 8, 128, 40)]


@pytest.mark.parametrize("heads, kv, dim, new", FORMS)
@pytest.mark.parametrize("size", [1e6, 1e7, 1e9, 1e20, 1e33])
def test_scores_of_any_size(heads, kv, dim, new, size):
    """One position's score is far above the others', wherever they lie: it alone is what comes out."""
    for n, best in ((30, 7), (700, 300), (1500, 1)):
        f = Filled([1], heads, kv, dim, 64, spare=1800, max_blocks=30)
        plan = f.cache.plan(f.slots, [n + new], at=[0])
        k, v = (torch.randn(n + new, kv, dim, generator=f.g, device="cuda").bfloat16() for _ in range(2))
        k[best] = 8.0
        f.cache.append(0, k, v, plan)
        plan = f.cache.plan(f.slots, [new], at=[n])
        f.cache.append(0, k[n:], v[n:], plan)
        q = ((1 + torch.rand(new, heads, dim, device="cuda", generator=f.g)) * size).bfloat16()
        want = stored(v[best]).repeat_interleave(heads // kv, 0)
        # one rounding to bf16, the stored value's own rounding to f16 (where it is left out), 16-bit weights
        assert ((f.cache.attention(0, q, plan).double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9).all()


@pytest.mark.parametrize("heads, kv, dim, new", FORMS)
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_queries_that_are_not_finite(heads, kv, dim, new, value):
    """Infinity times keys of one sign leaves scores of one sign: infinite all the same, whose softmax is not defined."""
    f = Filled([1], heads, kv, dim, 64, spare=1800, max_blocks=30)
    for n in (30, 700):
        plan = f.cache.plan(f.slots, [n + new], at=[0])
        k, v = (torch.randn(n + new, kv, dim, generator=f.g, device="cuda").bfloat16() for _ in range(2))
        k[:, :, 5] = 1.0
        f.cache.append(0, k, v, plan)
        f.k[0], f.v[0] = stored(k), stored(v)
        plan = f.cache.plan(f.slots, [new], at=[n])
        f.cache.append(0, k[n:], v[n:], plan)
        q = torch.randn(new, heads, dim, device="cuda", generator=f.g).bfloat16()
        want = f.want(q, [new])
        row, head = new // 2, heads - 1
        bad = q.clone()
        bad[row, head, 5] = value
        out = f.cache.attention(0, bad, plan)
        assert out[row, head].isnan().all()
        out[row, head] = want[0][row, head].bfloat16()
        close(out, want)


@pytest.mark.parametrize("heads, kv, dim, chunk", [(16, 8, 64, 200), (32, 8, 128, 70), (12, 4, 96, 30)])
def test_a_mixed_step_as_two_plans(heads, kv, dim, chunk):
    """A prompt's chunk and single tokens of other sequences in one step, a plan for each: the single tokens' bits are those of a step of
    their own, and both are right; as one plan too."""
    lens = [400, 37, 900, 1, 2100]
    outs = []
    for kind in ("two", "alone", "one"):
        f = Filled(lens, heads, kv, dim, 64, seed=8, spare=chunk)
        new = [1, 1, chunk, 1, 1]
        few = [i for i in range(5) if i != 2]
        k, v, q = (torch.randn(sum(new), h, dim, device="cuda", generator=f.g).bfloat16() for h in (kv, kv, heads))
        first = [0, 1, 2, 2 + chunk, 3 + chunk]
        rows = torch.tensor([first[i] for i in few], device="cuda")
        for i, m in enumerate(new):
            a = first[i]
            f.k[i], f.v[i] = torch.cat([f.k[i], stored(k[a:a + m])]), torch.cat([f.v[i], stored(v[a:a + m])])
        if kind == "one":
            plan = f.cache.plan(f.slots, new)
            f.cache.append(0, k, v, plan)
            close(f.cache.attention(0, q, plan), f.want(q, new))
            continue
        plans = [(f.cache.plan([f.slots[i] for i in few]), rows)]
        if kind == "two":
            plans.append((f.cache.plan([f.slots[2]], [chunk]), torch.arange(2, 2 + chunk, device="cuda")))
        out = torch.zeros_like(q)
        for plan, r in plans:
            f.cache.append(0, k[r], v[r], plan)
        for plan, r in plans:
            out[r] = f.cache.attention(0, q[r], plan)
        if kind == "two":
            close(out, f.want(q, new))
        outs.append(out[rows])
        f.cache.check_device()
    assert torch.equal(*outs)


@pytest.mark.parametrize("heads, kv, dim, new", [(32, 4, 64, 1), (16, 2, 96, 1), (26, 2, 128, 1), (12, 2, 96, 3), (4, 4, 64, 20), (16, 8, 64, 150), (12, 4, 96, 180),
                                                 (32, 8, 128, 40)])
def test_large_values_of_little_weight(heads, kv, dim, new):
    """Weights of 2^-15 to 2^-30 on values a million times the others': they are a part of the sum that is right to their own 11 bits."""
    f = Filled([1], heads, kv, dim, 64, spare=1300, max_blocks=30)
    for n in (60, 900):
        plan = f.cache.plan(f.slots, [n + new], at=[0])
        k, v = (torch.randn(n + new, kv, dim, generator=f.g, device="cuda") for _ in range(2))
        v *= 0.01
        k[5:n:9], v[5:n:9] = -2.0, v[5:n:9] * 2e6
        k, v = k.bfloat16(), v.clamp(-60000, 60000).bfloat16()
        f.cache.append(0, k, v, plan)
        f.k[0], f.v[0] = stored(k), stored(v)
        plan = f.cache.plan(f.slots, [new], at=[n])
        f.cache.append(0, k[n:], v[n:], plan)
        q = torch.randn(new, heads, dim, device="cuda", generator=f.g).abs().bfloat16()
        ref, mag, _ = f.want(q, [new])
        # weights below 2^-29 of the largest: half a unit of 2^-39 each
        close(f.cache.attention(0, q, plan), (ref, mag, 2.0 ** -40 * f.v[0].abs().sum(0).amax()))
