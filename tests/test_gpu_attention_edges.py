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
