"""The barrier protocol of the windowed attention kernels, explored on the CPU.

An mbarrier's wait tells neighbouring phases apart only (by parity), so every wait has to look before its barrier
can move on a second time, whatever the relative speed of the warps. The waits, arrivals and commits are read
from the kernels' source, with their barrier and parity expressions, and run here as small programs: the warp that
issues the products, two softmax warps, and the tensor core, which finishes products in order but may deliver the
arrivals of its commits in any order. Every interleaving of a few key tiles is tried: none may get stuck, read
scores or rescale an output before the product that makes them is done, or overwrite probabilities in use.
"""
import os
import re

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "r9700_stack_b200", "csrc", "window_attn.cu")

WAIT = re.compile(r"warp_wait\(&?(\w+)(?:\[(.+?)\])?, \(uint32_t\)\((.+)\), a\.timeout_ns\)")
COMMIT = re.compile(r"commit\(&?(\w+)(?:\[(.+?)\])?, go\)")
ARRIVE = re.compile(r"mbar_arrive\(&?(\w+)(?:\[(.+?)\])?\)")
COND = re.compile(r"if \(([^()]+)\) ok &= ")
NAMES = ("s_full", "s_free", "p_full", "pv_done")

# kernel: (where it begins, where it ends, the line that opens the rescale of O, the line after it)
KERNELS = {
    "dec": ("window_attn_dec_kernel(const", "Chunks: a tile of up to", "if (any) {", "uint8_t* prow"),
    "chunk": ("window_attn_chunk_kernel(const", "static void launch_cluster", "__any_sync(0xffffffffu, need)", "tmem_st_wait();"),
}


def _events(lines, rescale=(None, None)):
    """(kind, barrier, index expression, parity expression, condition, inside the rescale) of each line in order."""
    out, inside = [], False
    for line in lines:
        if rescale[0] and rescale[0] in line:
            inside = True
        elif rescale[1] and rescale[1] in line:
            if inside:
                out.append(("rescaled", "", "", "", "", False))
            inside = False
        for kind, pat in (("wait", WAIT), ("commit", COMMIT), ("arrive", ARRIVE)):
            m = pat.search(line)
            if m and m.group(1) in NAMES:
                cond = COND.search(line)
                out.append((kind, m.group(1), m.group(2) or "0", m.group(3) if kind == "wait" else "",
                            cond.group(1) if cond else "", inside))
    return out


def _kernel(name):
    begin, end, *rescale = KERNELS[name]
    with open(SRC) as f:
        text = f.read()
    text = text[text.index(begin):]
    text = text[: text.index(end)]
    mma = text[text.index("} else if (warp == 1) {"):]
    soft = mma[mma.index("\n  } else {"):]
    mma = mma[: mma.index("\n  } else {")]
    issue = mma[mma.index("auto issue_s"): mma.index("if (ok) ok = issue_s(0);")]
    loop = mma[mma.index("for (int j = 0; ok && j < n; ++j) {"):]
    soft = soft[soft.index("for (int j = 0; j < n; ++j) {"):]
    at = re.search(r"\n    \}\n", soft).start()  # the end of the loop over tiles
    tiles, after = _events(soft[:at].splitlines(), rescale), _events(soft[at:].splitlines())
    got = dict(issue=_events(issue.splitlines()), loop=_events(loop.splitlines()), tiles=tiles, after=after)
    assert [e[0] for e in got["issue"]].count("commit") == 1 and [e[0] for e in got["loop"]].count("commit") == 1
    assert any(e[0] == "rescaled" for e in tiles) and sum(e[0] == "arrive" and e[1] == "p_full" for e in tiles) == 1
    assert len(after) == 1
    return got


def _value(expr, j, n):
    expr = expr.replace("&&", " and ").replace("||", " or ")
    return int(eval(expr, {}, dict(j=j, n=n, s=j & 1, pb=j & 1)))  # noqa: S307 (the kernel's own index arithmetic)


def _program(events, j, n, product=None):
    out = []
    for kind, bar, idx, parity, cond, inside in events:
        if inside and j == 0:  # there is no output to rescale yet
            continue
        if kind == "rescaled":
            out.append(("check", "rescale", j))
            continue
        if cond and not _value(cond, j, n):
            continue
        key = (bar, _value(idx, j, n))
        if kind == "wait":
            out.append(("maybe" if inside else "wait", key, _value(parity, j, n)))
            if bar == "s_full":
                out.append(("check", "scores", j))
        elif kind == "commit":
            out += [("product", (product, j)), ("commit", key)]
        else:
            if bar == "p_full":
                out.append(("check", "probabilities", j))
            out.append(("arrive", key))
    return out


def _explore(k, n):
    """The first thing that goes wrong in some interleaving, or None."""
    mma = _program(k["issue"], 0, n, "S")
    for j in range(n):
        if j + 1 < n:
            mma += _program(k["issue"], j + 1, n, "S")
        mma += _program(k["loop"], j, n, "PV")
    soft = []
    for j in range(n):
        soft += _program(k["tiles"], j, n)
    soft += _program(k["after"], 0, n) + [("check", "output", n)]
    products = [e[1] for e in mma if e[0] == "product"]
    commits, made = [], 0  # (barrier, products before it)
    for e in mma:
        made += e[0] == "product"
        if e[0] == "commit":
            commits.append((e[1], made))
    bars = sorted({e[1] for e in mma + soft if e[0] in ("wait", "maybe", "commit", "arrive")})
    slot = {b: i for i, b in enumerate(bars)}
    need = [2 if b[0] in ("p_full", "s_free") else 1 for b in bars]  # arrivals of a phase: both softmax warps, or a commit
    issued = [[0, 0]]
    for e in mma:
        issued.append([issued[-1][0] + (e[0] == "product"), issued[-1][1] + (e[0] == "commit")])

    def arrive(state, b):
        phase, count = state[slot[b]]
        count += 1
        new = (phase + 1, 0) if count == need[slot[b]] else (phase, count)
        return state[: slot[b]] + (new,) + state[slot[b] + 1:]

    def passes(state, b, parity):
        return (state[slot[b]][0] & 1) != parity

    start = (0, (0, 0), (0, 0), 0, 0, tuple((0, 0) for _ in bars))  # mma, softmax (place, rescaling), done, fired, barriers
    seen, todo = {start}, [start]
    while todo:
        m, s0, s1, done, fired, st = todo.pop()
        nxt = []
        if m < len(mma):
            e = mma[m]
            if e[0] != "wait" or passes(st, e[1], e[2]):
                if e[0] == "product" and e[1][0] == "PV":  # the scores' and probabilities' reader
                    j = e[1][1]
                    for place, _ in (s0, s1):
                        if ("check", "probabilities", j) not in soft[:place]:
                            return f"PV({j}) issued before its probabilities"
                nxt.append((m + 1, s0, s1, done, fired, st))
        if done < issued[m][0]:
            nxt.append((m, s0, s1, done + 1, fired, st))
        for c in range(issued[m][1]):
            if not fired >> c & 1 and commits[c][1] <= done:
                nxt.append((m, s0, s1, done, fired | 1 << c, arrive(st, commits[c][0])))
        finished = set(products[:done])
        for w, (place, rescaling) in enumerate((s0, s1)):
            if place == len(soft):
                continue
            e, moves, new = soft[place], [], st
            if e[0] == "wait" and passes(st, e[1], e[2]):
                moves = [(place + 1, rescaling)]
            elif e[0] == "maybe":
                if not rescaling:
                    skip = next(i for i in range(place, len(soft)) if soft[i][:2] == ("check", "rescale"))
                    moves.append((skip + 1, 0))
                if passes(st, e[1], e[2]):
                    moves.append((place + 1, 1))
            elif e[0] == "arrive":
                new, moves = arrive(st, e[1]), [(place + 1, 0)]
            elif e[0] == "check":
                j = e[2]
                if e[1] == "scores" and ("S", j) not in finished:
                    return f"S({j}) read before it is done"
                if e[1] == "rescale" and rescaling and ("PV", j - 1) not in finished:
                    return f"O rescaled in tile {j} before PV({j - 1}) is done"
                if e[1] == "probabilities" and j >= 2 and ("PV", j - 2) not in finished:
                    return f"probabilities of tile {j} over those of a product that runs"
                if e[1] == "output" and ("PV", n - 1) not in finished:
                    return "output read before the last product is done"
                moves = [(place + 1, 0 if e[1] == "rescale" else rescaling)]
            for mv in moves:
                nxt.append((m, mv if w == 0 else s0, mv if w == 1 else s1, done, fired, new))
        if not nxt and (m < len(mma) or s0[0] < len(soft) or s1[0] < len(soft)):
            where = mma[m] if m < len(mma) else None
            return f"stuck: products {where}, softmax {[soft[p] if p < len(soft) else None for p, _ in (s0, s1)]}"
        for x in nxt:
            if x not in seen:
                seen.add(x)
                todo.append(x)
    return None


@pytest.mark.parametrize("name", ["dec", "chunk"])
@pytest.mark.parametrize("tiles", [1, 2, 3, 5])
def test_every_interleaving_ends_and_reads_what_is_done(name, tiles):
    assert _explore(_kernel(name), tiles) is None


def test_a_single_barrier_for_the_probabilities_is_found_out():
    """The oracle itself: with one p_full barrier whose parity turns every tile, the issuing warp can miss a phase."""
    k = _kernel("chunk")
    one = lambda e: (e[0], e[1], "0", "j & 1" if e[0] == "wait" else "", *e[4:]) if e[1] == "p_full" else e  # noqa: E731
    k = {part: [one(e) for e in events] for part, events in k.items()}
    assert "stuck" in (_explore(k, 4) or "")
