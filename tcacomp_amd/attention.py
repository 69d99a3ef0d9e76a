"""Operator programs of an attention sublayer over a paged cache: block tables
and slot maps, rotary positions, the same while keys and values are stored, and
attention (include/tca_op.h has the mathematics, the tensors of each and what
may overlap). They are operators as those of ``operators`` are:

    from tcacomp_amd import attention, compiler

    place = compiler.compile_program(attention.page_table())
    store = compiler.compile_program(attention.rotary_cache("bf16"))
    attend = compiler.compile_program(attention.paged_attention("bf16"))

    place.launch([held, new, free, first, table, starts, lens, pos, slot, next], free_dims=(page,))
    store.launch([x, pos, slot, freq, q, k, v], scalars=(1.0,))        # x [T, HK (G + 2), D]
    attend.launch([q, k, v, table, starts, lens, y], scalars=(D ** -0.5,))

A step of serving is these three launches whatever the lengths are, since those
stay on the GPU: captured once, they replay for every batch of the same extents.
The lists (the i32 tensors, freq and lse) may be slices of longer ones, of any
start; x, y, q, k and v are 16-byte aligned at theirs.
"""
from .operators import _listed, _make, Operator


def page_table():
    """held, new [S], free [F], first [1] -> table [S, P], starts [S + 1],
    lens [S], pos, slot [T], next [1], all i32; free dim page, the tokens of a
    page. The table's columns of held tokens are read, those of new ones
    stored; rows of pos and slot behind the last token are -1."""
    return Operator("page_table", "")


def rotary(elem, interleaved=False, inverse=False):
    """x [T, H, D], pos [T], freq [F] -> y [T, H, D]; scalar scale. The first 2 F
    of a head's D features are turned, in halves or (`interleaved`) as
    neighbours; `inverse` is the gradient. y may be x."""
    return _make("rotary", elem, interleaved=interleaved, inverse=inverse)


def rotary_cache(elem, interleaved=False):
    """x [T, HK (G + 2), D], pos, slot [T], freq [F] -> q [T, HK, G, D] and, where
    slot is not negative, the rows of k, v [PAGES, HK, PAGE, D]; scalar scale."""
    return _make("rotary_cache", elem, interleaved=interleaved)


def paged_attention(elem, window=False, stats=False):
    """q [T, HK, G, D], k, v [PAGES, HK, PAGE, D], table [S, P], starts [S + 1],
    lens [S] -> y [T, HK, G, D], (lse [T, HK, G]); scalar scale, with `window` a
    free dim: how many keys a query sees, its own among them."""
    return _make("paged_attention", elem, stats=stats, window=window)


def list_operators():
    """{operator: the attributes it takes}, of this module, as the library lists them."""
    return _listed(globals())


def all_builds():
    """(name, factory, emit flags) of every program that build() compiles."""
    made = [page_table]
    for e in ("f32", "bf16", "f16"):
        for inter in (False, True):
            made += [lambda e=e, i=inter, v=inverse: rotary(e, i, v) for inverse in (False, True)]
            made.append(lambda e=e, i=inter: rotary_cache(e, i))
    for e in ("bf16", "f16"):
        made += [lambda e=e, w=w, s=s: paged_attention(e, w, s) for w in (False, True) for s in (False, True)]
    return [("attention_%d" % i, f, 0) for i, f in enumerate(made)]
