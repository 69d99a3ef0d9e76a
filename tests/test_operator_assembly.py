"""The pipelined products of the operator programs, checked on their gfx950
assembly: their matrix instructions are inline asm, whose hazards the compiler
does not see, and their waits count the loads in flight by hand."""
import os
import re
import subprocess

import pytest

from test_abi_and_plan import REPO, _regs, _vgpr_writes
from tcacomp_amd import operators

PROGRAMS = {
    "linear": lambda: operators.linear("bf16", act="gelu", bias=True),
    "linear_backward": lambda: operators.linear_backward("f16", act="silu"),
    "gated": lambda: operators.gated("f16", act="silu", save=True),
    "gated_backward": lambda: operators.gated_backward("bf16", act="silu"),
}


def kernels(op, tmp_path):
    """{kernel: (template arguments, assembly)} of the kernels with a ring."""
    e = op.emit()
    src, asm = tmp_path / "k.hip", tmp_path / "k.s"
    src.write_text(e.source)
    flags = [f for f in e.hipcc if f != "--genco"]
    hipcc = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "bin", "hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    r = subprocess.run([hipcc] + flags + ["--cuda-device-only", "-S", "-o", str(asm), "-I",
                                          os.path.join(REPO, "tcacomp_amd", "csrc", "include"), str(src)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = asm.read_text().split("\n")
    found = {}
    for name, body in re.findall(r"(tca_\w+)\([^{]*\{(.*?)\n\}", e.source, re.S):
        m = re.search(r"product_ring<([^>]*)>", body)
        if not m:
            continue
        start = next(i for i, l in enumerate(lines) if l.startswith(name + ":"))
        end = next(i for i in range(start, len(lines)) if lines[i].startswith(".Lfunc_end"))
        code = [l.split(";")[0].rstrip() if not l.startswith(".L") else l.split(":")[0] + ":" for l in lines[start + 1:end]]
        args = [{"true": 1, "false": 0}.get(a.strip()) if a.strip() in ("true", "false") else int(a) for a in m.group(1).split(",")]
        found[name] = (args, [l.strip() for l in code if l.strip()])
    return found


class Flow:
    """Predecessors and successors of every instruction of one kernel."""

    def __init__(self, code):
        self.code = code
        labels = {l[:-1]: i for i, l in enumerate(code) if l.endswith(":")}
        self.next = [[] for _ in code]
        for i, l in enumerate(code):
            m = re.match(r"s_(c?)branch\S*\s+(\S+)$", l)
            assert not l.startswith(("s_setpc", "s_swappc", "s_call")), l
            if m:
                self.next[i].append(labels[m.group(2)])
            if not l.startswith("s_endpgm") and not (m and not m.group(1)) and i + 1 < len(code):
                self.next[i].append(i + 1)
        self.prev = [[] for _ in code]
        for i, to in enumerate(self.next):
            for j in to:
                self.prev[j].append(i)

    def back(self, start, stop):
        """The first instructions that `stop` holds for, on every way back from start."""
        seen, todo, hits = set(), list(self.prev[start]), set()
        while todo:
            i = todo.pop()
            if i in seen:
                continue
            seen.add(i)
            if stop(self.code[i]):
                hits.add(i)
            else:
                todo += self.prev[i]
        return hits

    def least(self, start, count, until):
        """The least `count`ed instructions between start and an earlier one
        that `until` holds for, over every way back (None: none is met)."""
        best, todo, found = {start: 0}, [start], None
        while todo:
            i = todo.pop(0)
            for j in self.prev[i]:
                if until(self.code[j]):
                    found = best[i] if found is None else min(found, best[i])
                    continue
                n = best[i] + (1 if count(self.code[j]) else 0)
                if j not in best or n < best[j]:
                    best[j] = n
                    todo.append(j)
        return found


def in_flight(qa, qb, sa, sb):
    """Loads that may be in flight at a turn's barrier: those issued after the
    last one of the next turn's, over enough turns, the order written out."""
    issued, least = [], None
    for t in range(max(sa - 1, sb)):
        issued += [t] * qa if t < sa - 1 else []
        issued += [t] * qb if t < sb else []
    for t in range(32):
        issued += [t + sa - 1] * qa
        last = max(i for i, j in enumerate(issued) if j == t + 1)
        n = len(issued) - 1 - last
        least = n if least is None else min(least, n)
        issued += [t + sb] * qb
    return least


@pytest.fixture(scope="module", params=sorted(PROGRAMS))
def rings(request, tmp_path_factory):
    found = kernels(PROGRAMS[request.param](), tmp_path_factory.mktemp("asm"))
    assert len(found) >= 5
    return found


def loops(code):
    """(first, last) of the innermost loops that hold matrix instructions."""
    labels = {l[:-1]: i for i, l in enumerate(code) if l.endswith(":")}
    spans = []
    for i, l in enumerate(code):
        m = re.match(r"s_c?branch\S*\s+(\S+)$", l)
        if m and labels[m.group(1)] <= i and any(c.startswith("v_mfma") for c in code[labels[m.group(1)]:i]):
            spans.append((labels[m.group(1)], i))
    return [s for s in spans if not any(o != s and s[0] <= o[0] and o[1] <= s[1] for o in spans)]


def mentions_agpr(line):
    return re.search(r"\ba(\[\d|\d)", line) is not None


def test_matrix_instructions_and_their_hazards(rings):
    """Accumulators stay in AGPRs in place; an operand comes from LDS reads
    only, on every way to the instruction; two s_nop 7 between the accumulators'
    start and the first product, three between the last and the first read."""
    for name, (_, code) in rings.items():
        flow = Flow(code)
        mfma = [i for i, l in enumerate(code) if l.startswith("v_mfma")]
        assert len(mfma) >= 32, name
        for i in mfma:
            ops = [o.strip() for o in code[i].split(None, 1)[1].split(",")]
            assert ops[0] == ops[3] and ops[0].startswith("a["), code[i]
            for op in ops[1:3]:
                kind, regs = _regs(op)
                assert kind == "v", code[i]
                for r in regs:
                    writers = flow.back(i, lambda l: r in _vgpr_writes(l))
                    assert writers and all(code[w].startswith("ds_read") for w in writers), (name, code[i], [code[w] for w in writers])
        nop = lambda l: l == "s_nop 7"  # noqa: E731
        others = [i for i, l in enumerate(code) if mentions_agpr(l) and not l.startswith("v_mfma")]
        writes = [i for i in others if code[i].startswith("v_accvgpr_write")]
        assert writes, name
        for i in mfma:
            n = flow.least(i, nop, lambda l: l.startswith("v_accvgpr_write"))
            assert n is None or n >= 2, (name, n)
        for i in others:
            n = flow.least(i, nop, lambda l: l.startswith("v_mfma"))
            assert n is None or n >= 3, (name, code[i], n)


def test_loops_wait_for_the_counted_loads_only(rings):
    """Each of the two loops has its turn's loads, one barrier, one wait on
    loads, for exactly as many as may be in flight, and no spill that would
    share the counter."""
    for name, (args, code) in rings.items():
        bm, hb, wgm, wgn, sa, sb = args[-6:]
        waves = wgm * wgn
        qa, qb = bm // 8 // waves, 2 * hb // 8 // waves
        assert not [l for l in code if "scratch_" in l], name
        found = loops(code)
        assert len(found) == 2, (name, found)
        for first, last in found:
            body = code[first:last + 1]
            assert sum(l.startswith("v_mfma") for l in body) == 2 * (bm // wgm // 16) * (2 * hb // wgn // 16), name
            assert not [l for l in body if "accvgpr" in l], name
            assert sum(l.startswith("s_barrier") for l in body) == 1, name
            # every load into LDS is issued whatever its address: none is branched round
            loads = [l for l in body if "load_lds" in l]
            assert len(loads) == qa + qb and not [l for l in body[:-2] if l.startswith("s_cbranch")], (name, len(loads))
            others = [l for l in body if l.startswith(("global_load", "buffer_load", "flat_load")) and "load_lds" not in l]
            assert not others, (name, others[:3])
            waits = [int(m.group(1)) for l in body for m in [re.search(r"vmcnt\((\d+)\)", l)] if m]
            assert waits == [in_flight(qa, qb, sa, sb)], (name, waits, in_flight(qa, qb, sa, sb))
