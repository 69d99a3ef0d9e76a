"""The attention operators on the GPU where a caller's tensors are not the usual
ones: lists that are slices of longer ones, batches shorter than the new tokens,
pages of no tokens, lengths that leave the batch, and values that are not finite
in tiles that lie anywhere in a workgroup's run."""
import random

import pytest
import torch

import attention_ref as ref
from operators_ref import DTYPES
from tcacomp_amd import attention
from test_gpu_attention import ints, launch_page_table, make, run
from test_gpu_operators import close, gen_of, program, rand

pytestmark = pytest.mark.gpu


# ------------------------------------------------- lists that start anywhere

def sliced(t, by):
    """A copy of t that starts `by` elements into a longer buffer, and that buffer's
    elements around it, with their values."""
    n = t.numel()
    buf = torch.full((n + 8,), -77, device="cuda", dtype=t.dtype)
    buf[by:by + n] = t.reshape(-1)
    return buf[by:by + n].view(t.shape), [buf[:by], buf[by + n:]]


def launch_sliced(p, tensors, lists, by, **how):
    """The launch with the named tensors as slices; all of its tensors, after a check
    that nothing around the slices was written."""
    around, moved = [], []
    for i, t in enumerate(tensors):
        if i in lists:
            t, rest = sliced(t, by)
            assert t.data_ptr() % 16 == 4 * by % 16
            around += rest
        else:
            t = t.clone()
        moved.append(t)
    p.launch(moved, **how)
    assert all((r == -77).all() for r in around)
    return moved


@pytest.mark.parametrize("by", [1, 2, 3])
def test_lists_that_are_slices(gpu, by):
    g = gen_of("slices", by)
    f = torch.rand(32, generator=g, device="cuda")
    table = torch.arange(60, device="cuda", dtype=torch.int32).view(6, 10)
    x, y = rand(g, (9, 4, 64), "bf16"), torch.zeros((9, 4, 64), device="cuda", dtype=torch.bfloat16)
    k, v, q = rand(g, (7, 1, 16, 64), "bf16"), rand(g, (7, 1, 16, 64), "bf16"), torch.zeros((9, 1, 2, 64), device="cuda", dtype=torch.bfloat16)
    pos, slot = ints(list(range(9))), torch.randperm(112, generator=g, device="cuda")[:9].int()
    a = make(gen_of("sliced attention"), "bf16", [700, 300, 40], [90, 1, 3], 2, 4, 64, 16)
    aq, ak, av, at, starts, lens = a
    lists = [
        (program(attention.page_table), [ints([5, 0, 33, 16, 2, 9]), ints([30, 1, 0, 16, 7, 1]), ints(range(100, 131)), ints([2]), table, ints([0] * 7), ints([0] * 6),
                                         ints([0] * 57), ints([0] * 57), ints([0])], range(10), dict(free_dims=(16,))),
        (program(attention.rotary, "bf16"), [x, pos, f, y], (1, 2), dict(scalars=(1.0,))),
        (program(attention.rotary, "f32", True), [x.float(), pos, f, y.float()], (1, 2), dict(scalars=(1.0,))),
        (program(attention.rotary_cache, "bf16"), [x, pos, slot, f, q, k, v], (1, 2, 3), dict(scalars=(1.0,))),
        (program(attention.paged_attention, "bf16", False, True),
         [aq, ak, av, at, ints(starts), ints(lens), torch.zeros_like(aq), torch.zeros(aq.shape[:3], device="cuda")], (3, 4, 5, 7), dict(scalars=(0.125,))),
    ]
    for p, tensors, which, how in lists:
        print(p.name, by, flush=True)
        want = launch_sliced(p, tensors, (), 0, **how)
        for got, w in zip(launch_sliced(p, tensors, set(which), by, **how), want):
            assert torch.equal(got.nan_to_num(3.0), w.nan_to_num(3.0)), p.name


# ------------------------------------- batches shorter than the new tokens

@pytest.mark.parametrize("S,new,page,columns,keep", [
    (1, 40, 16, 4, 0.5), (1, 40, 16, 4, 0.0), (7, 40, 24, 5, 0.3), (64, 1, 16, 70, 0.6), (300, 9, 1, 30, 0.01), (1500, 30, 16, 4, 0.4), (3, 6000, 64, 100, 0.7)])
def test_page_table_of_a_short_batch(gpu, S, new, page, columns, keep):
    """Tokens from T on are in neither pos nor slot; the table's columns, starts, lens
    and the next free page are those of all new tokens."""
    print("short table", S, new, page, keep, flush=True)
    rng = random.Random(S * 100 + page)
    fresh = [rng.choice((0, 1, new, rng.randint(0, new))) for _ in range(S)]
    fresh[S // 2] = new
    held = [rng.randint(0, columns * page - 1) for _ in range(S)]
    ids = list(range(S * columns + 9))
    rng.shuffle(ids)
    table, at = [], 0
    for h in held:
        n = -(-h // page)
        table.append(ids[at:at + n] + [-5] * (columns - n))
        at += n
    free = ids[at:at + max(1, sum(-(-n // page) for n in fresh) - 1)]
    T = int(sum(fresh) * keep)
    got = launch_page_table(held, fresh, free, 1, table, page, T)
    want = ref.page_table(held, fresh, free, 1, table, page, sum(fresh))
    for g, w, what in zip(got, want, ("table", "starts", "lens", "pos", "slot", "next")):
        assert g == ([w] if what == "next" else w[:T] if what in ("pos", "slot") else w), what


def whole(elem, case, scale, window=0):
    """attention_ref.paged_attention of a case whose starts go past its rows: of a batch
    that has them all, cut to the rows that are there."""
    q, k, v, table, starts, lens = case
    T = q.shape[0]
    rest = torch.zeros((max(starts[-1] - T, 0),) + q.shape[1:], device=q.device, dtype=q.dtype)
    return [t[:T] for t in ref.paged_attention(torch.cat([q, rest]), k, v, table, starts, lens, scale, window, DTYPES[elem])]


def agree(y, lse, want, rows=slice(None)):
    """Values within their bounds; NaN (of rows that see it) and -inf in the same places."""
    y, lse, (wy, wl, by, bl) = y[rows], lse[rows], (t[rows] for t in want)
    none = wl == -float("inf")
    assert torch.equal(none, lse == -float("inf")) and torch.equal(wy.isnan(), y.isnan()) and torch.equal(wl.isnan(), lse.isnan())
    odd, wild = wy.isnan(), none | wl.isnan()
    close(torch.where(odd, 0.0, y), torch.where(odd, 0.0, wy), torch.where(odd, 1.0, by), "y")
    close(torch.where(wild, 0.0, lse), torch.where(wild, 0.0, wl), torch.where(wild, 1.0, bl), "lse")


@pytest.mark.parametrize("elem", ["bf16", "f16"])
@pytest.mark.parametrize("lens,fresh,G,D,T,window", [
    ([100], [10], 4, 64, 3, 0), ([700, 90], [300, 30], 4, 64, 310, 0), ([700, 90], [300, 30], 2, 128, 170, 0), ([50, 50, 50], [20, 20, 20], 1, 256, 25, 0),
    ([3000, 40], [6, 8], 4, 128, 9, 0), ([900, 800], [400, 300], 2, 64, 500, 33)])
def test_attention_of_a_short_batch(gpu, elem, lens, fresh, G, D, T, window):
    """Rows keep the positions that starts and lens give them, whether the batch has the rows behind them or not."""
    print("short batch", lens, fresh, T, flush=True)
    q, k, v, table, starts, lens = make(gen_of("cut", T, D, elem), elem, lens, fresh, 2, G, D, 16)
    case = (q[:T].contiguous(), k, v, table, starts, lens)
    y, lse = run(elem, case, D ** -0.5, window)
    agree(y, lse, whole(elem, case, D ** -0.5, window))


def test_a_step_of_a_short_batch(gpu):
    """Tables, stores and attention of a batch with room for some of the new tokens
    only: its rows are those of a batch with room for all, no page is lost, and a
    sequence that was there as a whole goes on."""
    S, HK, G, D, page, columns = 3, 2, 4, 64, 16, 8
    g = gen_of("short step")
    freq = torch.rand(D // 2, generator=g, device="cuda")
    fresh, T = [30, 50, 21], 62  # all of the first sequence, some of the second, none of the third
    x = rand(g, (sum(fresh), HK * (G + 2), D), "bf16")
    free = torch.randperm(S * columns, generator=g, device="cuda").int()

    class State:
        def __init__(self):
            self.table = torch.full((S, columns), -1, device="cuda", dtype=torch.int32)
            self.k, self.v = (torch.full((S * columns, HK, page, D), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2))
            self.held, self.first = ints([0] * S), ints([0])

        def step(self, new, x):
            T = x.shape[0]
            starts, lens, pos, slot, after = ints([0] * (S + 1)), ints([0] * S), ints([0] * T), ints([0] * T), ints([0])
            q = torch.zeros((T, HK, G, D), device="cuda", dtype=x.dtype)
            y, lse = torch.full_like(q, -12345.0), torch.zeros((T, HK, G), device="cuda")
            program(attention.page_table).launch([self.held, ints(new), free, self.first, self.table, starts, lens, pos, slot, after], free_dims=(page,))
            program(attention.rotary_cache, "bf16").launch([x, pos, slot, freq, q, self.k, self.v], scalars=(1.0,))
            program(attention.paged_attention, "bf16", False, True).launch([q, self.k, self.v, self.table, starts, lens, y, lse], scalars=(D ** -0.5,))
            want = whole("bf16", (q, self.k, self.v, self.table, starts.tolist(), lens.tolist()), D ** -0.5)
            self.held, self.first = lens, after
            return q, y, lse, want

    full, short = State(), State()
    q, _, _, want = full.step(fresh, x)
    q2, y, lse, _ = short.step(fresh, x[:T].contiguous())
    assert torch.equal(q2, q[:T])
    for name in ("table", "held", "first"):
        assert torch.equal(getattr(short, name), getattr(full, name)), name
    agree(y, lse, [w[:T] for w in want])
    more = rand(g, (5, HK * (G + 2), D), "bf16")
    _, _, _, want = full.step([5, 0, 0], more)
    _, y, lse, _ = short.step([5, 0, 0], more)
    agree(y, lse, want)


def test_starts_and_lengths_that_leave_the_batch(gpu):
    """Against the rows that are there, between guards that nothing writes; of a cache
    whose rows past the sequences hold NaN, and of one that is finite."""
    q, k, v, table, _, _ = make(gen_of("leave"), "bf16", [100, 100, 100], [1, 1, 1], 2, 4, 64, 16)
    for k, v in ((k, v), (k.nan_to_num(0.5), v.nan_to_num(-0.25))):
        leave_the_batch(q, k, v, table)


def leave_the_batch(q, k, v, table):
    T, guard = 3, 2
    cases = [  # starts, lens; the same with starts inside, as the reference takes them: (starts, lens, rows to check)
        ([0, 2, 1, 900], [100, -5, 100], None, [0]),
        ([-3, 2, 2, 2], [100, 100, 100], ([0, 2, 2, 2], [100, 100, 100]), [0, 1]),
        ([-(1 << 31), 2, 2, 3], [100, 100, 77], ([0, 2, 2, 3], [100, 100, 77]), [0, 1, 2]),
        ([0, 2, 2, 3], [1 << 20, 5, (1 << 31) - 1], ([0, 2, 2, 3], [1 << 20, 5, (1 << 31) - 1]), [0, 1, 2]),
        ([0, 1, 3, 3], [1, -(1 << 31), 8], ([0, 1, 3, 3], [1, 0, 8]), [0, 1, 2]),
        ([2, 1, 0, 0], [100, 100, 100], ([0, 0, 0, 0], [0, 0, 0]), []),
        ([3, (1 << 31) - 1, 5, 9], [100, 100, 100], ([0, 0, 0, 0], [0, 0, 0]), []),
        ([0, 1, 1, 900], [100, -5, 1000], ([0, 1, 1, 900], [100, 0, 1000]), [0, 1, 2]),
    ]
    for starts, lens, inside, rows in cases:
        print(starts, lens, flush=True)
        y = torch.full((T + 2 * guard,) + q.shape[1:], -12345.0, device="cuda", dtype=q.dtype)
        lse = torch.full((T + 2 * guard,) + q.shape[1:3], -12345.0, device="cuda")
        program(attention.paged_attention, "bf16", False, True).launch(
            [q, k, v, table, ints(starts), ints(lens), y[guard:guard + T], lse[guard:guard + T]], scalars=(0.125,))
        for t in (y, lse):
            assert (t[:guard] == -12345.0).all() and (t[guard + T:] == -12345.0).all()
        y, lse = y[guard:guard + T], lse[guard:guard + T]
        if inside is None:  # row 1 is either sequence's; row 2 lies 798 before the third sequence's first key
            want = ref.paged_attention(q, k, v, table, [0, 2, 2, 2], [100, 0, 0], 0.125, 0, DTYPES["bf16"])
            assert (y[2] == 0).all() and (lse[2] == -float("inf")).all()
            assert ((y[1] == 0).all() and (lse[1] == -float("inf")).all()) or ((y[1].double() - want[0][1]).abs() <= want[2][1]).all()
        else:
            want = whole("bf16", (q, k, v, table, *inside), 0.125)
        agree(y, lse, want, rows)
        left = [r for r in range(T) if r not in rows] if inside is not None else []
        assert (y[left] == -12345.0).all() and (lse[left] == -12345.0).all()


def test_no_sequences_and_no_columns(gpu):
    """No sequence at all leaves every row; a table without columns hides every key."""
    q, k, v, table, starts, lens = make(gen_of("none"), "bf16", [40, 90], [3, 40], 2, 4, 64, 16)
    y, lse = run("bf16", (q, k, v, table[:0], [0], []), 0.125)
    assert (y == -12345.0).all() and (lse == -12345.0).all()
    y, lse = run("bf16", (q, k, v, table[:, :0].contiguous(), starts, lens), 0.125)
    assert (y == 0).all() and (lse == -float("inf")).all()


def test_the_largest_batch_of_the_allocation_free_launch(gpu):
    """512 (min(T, 32) + T) (4 D + 8) bytes and 16 KiB of its 32 MiB."""
    from tcacomp_amd import _lib
    for T, D, fits in ((93, 128, True), (94, 128, False), (31, 256, True), (32, 256, False)):
        case = make(gen_of("fits", T, D), "bf16", [2000], [T], 2, 1, D, 16)
        y, lse = run("bf16", case, D ** -0.5)
        agree(y, lse, whole("bf16", case, D ** -0.5))
        if fits:
            y2, lse2 = run("bf16", case, D ** -0.5, noalloc=True)
            assert torch.equal(y, y2) and torch.equal(lse, lse2)
        else:
            with pytest.raises(_lib.TcaError, match="scratch"):
                run("bf16", case, D ** -0.5, noalloc=True)


def test_pages_of_no_tokens(gpu):
    """A cache [9, 2, 0, 64]: no slot lies in it, no key is seen; queries are turned as ever."""
    g = gen_of("page 0")
    x, pos, freq = rand(g, (5, 8, 64), "bf16"), ints([3, 1, 4, 1, 5]), torch.rand(32, generator=g, device="cuda")
    outs = []
    for page, slot in ((0, [0, 1, 7, 1 << 30, 8]), (16, [-1] * 5)):
        q = torch.zeros((5, 2, 2, 64), device="cuda", dtype=torch.bfloat16)
        k, v = (rand(g, (9, 2, page, 64), "bf16") for _ in range(2))
        program(attention.rotary_cache, "bf16").launch([x, pos, ints(slot), freq, q, k, v], scalars=(1.0,))
        outs.append(q)
    assert torch.equal(outs[0], outs[1]) and outs[0].any()
    k = torch.zeros((9, 2, 0, 64), device="cuda", dtype=torch.bfloat16)
    for starts in ([0, 5], [0, 1]):
        y, lse = run("bf16", (outs[0], k, k.clone(), ints([[0, 1, 2]]), starts, [40]), 0.125)
        n = starts[1]
        assert (y[:n] == 0).all() and (lse[:n] == -float("inf")).all() and (y[n:] == -12345.0).all() and (lse[n:] == -12345.0).all()


# ------------------- values that are not finite, anywhere in a workgroup's run

def units(lens, fresh, HK, G, D, window=0):
    """(many, few): units of work of each kind, as the kernels count them."""
    most, many, few = (256, 0, 0) if D <= 128 else (128, 0, 0)
    keys_few = 256 if D <= 128 else 128
    heads = min(G, most)
    for L, n in zip(lens, fresh):
        if n == 0:
            continue
        big = n * G > 32
        step, block = (most // heads, 64) if big else (n, keys_few)
        total = 0
        for t0 in range(0, n, step):
            hi, lo = L - n + min(n, t0 + step), max(0, L - n + t0 + 1 - window) if window else 0
            total += max(1, (hi - 1) // block + 1 - lo // block if hi > lo else 0)
        total *= HK * (-(-G // heads) if big else 1)
        many, few = (many + total, few) if big else (many, few + total)
    return many, few


SHORT = [33 + 7 * i % 30 for i in range(150)]  # tiles of one block each
ODD = {  # lengths, new tokens, key heads, group, features, window, (sequence, place among its new tokens), units of a workgroup at least (many, few)
    "prompt": ([2500], [2500], 2, 1, 64, 0, [(0, 1203)], (2, 0)),
    "prompt f": ([1700, 33], [1700, 33], 2, 4, 128, 0, [(0, 700)], (3, 0)),
    "wide": ([1500, 300], [1500, 200], 2, 2, 256, 0, [(0, 800), (1, 3)], (3, 0)),
    "window": ([4000], [3000], 2, 2, 64, 300, [(0, 1501)], (2, 0)),
    "short ones": (SHORT, SHORT, 6, 1, 64, 0, [(76, 20)], (4, 0)),
    "short beside long": ([2100] + SHORT, [2100] + SHORT, 3, 2, 64, 0, [(0, 1000), (41, 17), (149, 30)], (6, 0)),
    "few": ([9000, 5000], [4, 7], 8, 4, 128, 0, [(0, 2), (1, 3)], (0, 2)),
    "few f": ([9001], [6], 2, 5, 64, 0, [(0, 3)], (0, 1)),
    "few wide": ([7000, 3000, 50], [3, 1, 8], 4, 4, 192, 0, [(0, 1), (2, 4)], (0, 1)),
    "few window": ([9000, 4000], [4, 8], 8, 4, 64, 3500, [(0, 1)], (0, 1)),
    "both": ([5000, 1900, 3000, 60], [5, 1000, 1, 60], 4, 4, 128, 0, [(0, 2), (1, 500)], (4, 1)),
}


@pytest.mark.parametrize("name", sorted(ODD))
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_values_that_are_not_finite_in_any_tile(gpu, name, bad):
    """A value of one key head of a new token: rows before it, rows whose window has left
    it, other heads and other sequences are as without it."""
    lens, fresh, HK, G, D, window, where, (many, few) = ODD[name]
    elem = "f16" if name.endswith("f") else "bf16"
    print(name, bad, elem, flush=True)
    counted = units(lens, fresh, HK, G, D, window)
    assert -(-counted[0] // 256) >= many and -(-counted[1] // 256) >= few, counted
    case = make(gen_of("any tile", name), elem, lens, fresh, HK, G, D, 16, pad=1)
    q, k, v, table, starts, _ = case
    want = ref.paged_attention(*case, D ** -0.5, window, DTYPES[elem])  # without them
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    for s, i in where:
        at, h = lens[s] - fresh[s] + i, (s + i) % HK
        v[int(table[s, at // 16]), h, at % 16, D // 2] = float(bad)
        last = fresh[s] if not window else min(fresh[s], i + window)
        hit[starts[s] + i:starts[s] + last, h] = True
    y, lse = run(elem, case, D ** -0.5, window)
    n = starts[-1]
    assert (y[n:] == -12345.0).all() and (lse[n:] == -12345.0).all()
    free = ~hit[:n]
    close(y[:n][free], want[0][:n][free], want[2][:n][free], "rows that do not see it")
    close(lse[:n], want[1][:n], want[3][:n], "the statistics, which no value enters")
    column = y[:n, :, :, D // 2][hit[:n]]
    assert column.isnan().all() if bad == "nan" else (column == float("inf")).all()
    rest = torch.ones(D, dtype=torch.bool, device="cuda")
    rest[D // 2] = False
    close(y[:n][hit[:n]][..., rest], want[0][:n][hit[:n]][..., rest], want[2][:n][hit[:n]][..., rest], "other columns of rows that see it")


def spoil(case, s, i, h, d, value):
    """Puts a value of new token i of sequence s, key head h, column d (or all) into the cache."""
    _, _, v, table, starts, lens = case
    at = lens[s] - (starts[s + 1] - starts[s]) + i
    page = case[1].shape[2]
    v[int(table[s, at // page]), h, at % page, d] = value


@pytest.mark.parametrize("elem", ["bf16", "f16"])
@pytest.mark.parametrize("D", [128, 256])
def test_infinite_values_before_nan(gpu, elem, D):
    """Rows between an infinite value and a NaN of the same column see the first alone,
    those behind both have NaN; -inf and inf make NaN where both are seen."""
    n = 300
    case = make(gen_of("inf nan", D, elem), elem, [n + 37], [n], 2, 2, D, 16)
    for i, d, value in ((20, 3, "inf"), (40, 3, "nan"), (50, 5, "-inf"), (90, 5, "inf"), (100, 7, "nan"), (270, 7, "inf"), (0, 9, "-inf"), (299, 9, "nan")):
        spoil(case, 0, i, 1, d, float(value))
    y, lse = run(elem, case, D ** -0.5)
    want, wl, by, bl = ref.paged_attention(*case, D ** -0.5, 0, DTYPES[elem])
    close(lse, wl, bl, "the statistics, which no value enters")
    for d, spans in ((3, ((0, 20, None), (20, 40, "inf"), (40, n, "nan"))), (5, ((0, 50, None), (50, 90, "-inf"), (90, n, "nan"))),
                     (7, ((0, 100, None), (100, n, "nan"))), (9, ((0, 299, "-inf"), (299, n, "nan")))):
        for a, b, value in spans:
            got = y[a:b, 1, :, d]
            if value == "nan":
                assert got.isnan().all(), (d, a)
            elif value:
                assert (got == float(value)).all(), (d, a)
            else:
                # the reference's products of 0 and what is not finite are NaN: without it
                clean = [t.clone() if t is case[2] else t for t in case]
                clean[2] = clean[2].nan_to_num(0.0, 0.0, 0.0)
                cy, _, cb, _ = ref.paged_attention(*clean, D ** -0.5, 0, DTYPES[elem])
                close(got, cy[a:b, 1, :, d], cb[a:b, 1, :, d], "rows before it")
    rest = torch.ones(D, dtype=torch.bool, device="cuda")
    rest[[3, 5, 7, 9]] = False
    close(y[..., rest], want[..., rest], by[..., rest], "other columns")
    close(y[:, 0], want[:, 0], by[:, 0], "the other head")


@pytest.mark.parametrize("window", [0, 40, 700])
def test_a_sequence_of_nan(gpu, window):
    """One of three sequences holds nothing but NaN values: its rows are NaN, the others as without it."""
    case = make(gen_of("all nan", window), "bf16", [900, 1300, 500], [300, 1000, 4], 2, 4, 64, 16)
    want = ref.paged_attention(*case, 0.125, window, DTYPES["bf16"])
    q, k, v, table, starts, _ = case
    v[table[1][table[1] >= 0].long()] = float("nan")
    y, lse = run("bf16", case, 0.125, window)
    mine = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    mine[starts[1]:starts[2]] = True
    assert y[mine].isnan().all()
    close(y[~mine], want[0][~mine], want[2][~mine], "the others")
    close(lse, want[1], want[3], "the statistics")


def test_values_that_are_not_finite_cost_little(gpu):
    """A prompt with a NaN at its first token or in all of them: a launch takes not many
    times as long as without (each row that saw one went through its keys again, by
    itself: 130 times). Rows of a tile that do not see a NaN of its do that still."""
    def took(case):
        q, k, v, table, starts, lens = case
        p = program(attention.paged_attention, "bf16")
        tensors = [q, k, v, table, ints(starts), ints(lens), torch.empty_like(q)]
        best = float("inf")
        for i in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            p.launch(tensors, scalars=(0.1,))
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b)) if i else best
        return best
    n = 4096
    case = make(gen_of("cost"), "bf16", [n], [n], 8, 4, 128, 64)
    clean = took(case)
    for what, tokens, most in (("first", [0], 12), ("all", range(n), 12)):
        spoilt = [t.clone() if t is case[2] else t for t in case]
        for i in (tokens if what != "all" else ()):
            spoil(spoilt, 0, i, slice(None), slice(None), float("nan"))
        if what == "all":
            spoilt[2].fill_(float("nan"))
        t = took(spoilt)
        print("NaN at %s: %.3f ms, %.3f without" % (what, t, clean), flush=True)
        assert t <= most * clean
