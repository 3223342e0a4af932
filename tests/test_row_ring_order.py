"""The order between the passes and the helpers of the row-loss ring kernel (CPU): every interleaving of a model.

In ``csrc/rowkernel.cuh`` the warps of the passes and the helper warps of a CTA hand a row's base, the
passes' states and the gradient's coefficients to each other through one place per helper, guarded by mbarriers.
The model has the same steps and barriers, with the layouts read from the source, and walks
through every order in which warps and helpers can take their steps: nobody may read what belongs to another row, and
nobody may be left waiting (in the kernel that wait runs into its limit and the row's gradient is missing).

The steps, for row i with helper h = i mod helpers:
    helper   base[h] = i, arrive ready[h] | wait states[h], read the states, coef[h] = i, arrive done[h] |
             the next row's base | lists: wait written[h], write the entries
    passes   first(i):  wait ready[h], read base[h], (forward only: wait done[h] of the row before) write the state,
                        arrive states[h]
             second(i): wait done[h], read coef[h], (lists, and with saved statistics: arrive written[h])
and with saved statistics the helper waits for written[h] of its row before instead of states[h].
"""

import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ferrite-tpu_b200", "csrc", "rowkernel.cuh")
WARPS, ROWS = 2, 5


def _value(text, lists, grad):
    m = re.fullmatch(r"\s*(.+) \? (.+?) : (.+)", text)
    names = {"LIST": lists, "GRAD": grad, "false": False, "true": True}
    if m:
        text = m.group(2) if eval(m.group(1).replace("||", "or"), names) else m.group(3)
    return eval(text, names)  # a number, or a product of numbers


def layouts():
    """(name, lists, grad, helpers, lag) of every layout in the source."""
    src = open(SOURCE).read()
    names = re.search(r"template <([^>]*)>\nstruct Layout", src).group(1)
    at = {n.split()[-1]: i for i, n in enumerate(names.split(","))}
    out = []
    for name, args in re.findall(r"^using (\w+) = Layout<(.*)>;", src, re.M):
        for lists in (False, True):
            for grad in (False, True):
                v = [_value(a, lists, grad) for a in args.split(",")]
                out.append((name, lists, grad, v[at["HELPERS"]], v[at["LAG"]] > 0))
    return out


def passes(i, kind, lists, helpers):
    """The steps of one warp for its pass over row i: ("wait", barrier, parity), ("read", place, row), ..."""
    h, turn = i % helpers, i // helpers % 2
    if kind == "first":
        return [("wait", f"ready{h}", turn), ("read", f"base{h}", i), ("state", h, i), ("arrive", f"states{h}")]
    if kind == "forward":
        return passes(i, "first", lists, helpers)[:2] + [("wait", f"done{h}", turn ^ 1), ("state", h, i), ("arrive", f"states{h}")]
    return [("wait", f"done{h}", turn), ("read", f"coef{h}", i)] + ([("arrive", f"written{h}")] if lists or kind == "saved" else [])


def programs(grad, saved, lag, lists, helpers):
    """The steps of a warp of the passes, and of each helper."""
    warp, behind = [], None
    for i in range(ROWS):
        if saved:
            warp += passes(i, "saved", lists, helpers)
            continue
        warp += passes(i, "first" if grad else "forward", lists, helpers)
        due = behind if lag else i
        if grad and due is not None:
            warp += passes(due, "second", lists, helpers)
        behind = i
    if grad and lag and not saved:
        warp += passes(behind, "second", lists, helpers)
    helper = []
    for h in range(helpers):
        rows = list(range(h, ROWS, helpers))
        p = [] if saved or not rows else [("write", f"base{h}", rows[0]), ("arrive", f"ready{h}")]
        for turn, i in enumerate(rows):
            if saved:
                p += [("wait", f"written{h}", turn % 2 ^ 1)]
            else:
                p += [("wait", f"states{h}", turn % 2), ("merge", h, i)]
            p += [("write", f"coef{h}", i), ("arrive", f"done{h}")]
            if not saved and turn + 1 < len(rows):
                p += [("write", f"base{h}", rows[turn + 1]), ("arrive", f"ready{h}")]
            if lists and grad:
                p += [("wait", f"written{h}", turn % 2)]
        helper.append(p)
    return [list(warp) for _ in range(WARPS)] + helper


def faults(progs):
    """Walks every interleaving; the first thing that goes wrong, or None."""
    names = sorted({s[1] for p in progs for s in p if s[0] in ("wait", "arrive")})
    count = {n: 1 if n.startswith(("ready", "done")) else WARPS for n in names}
    bar = {n: i for i, n in enumerate(names)}
    places = sorted({s[1] for p in progs for s in p if s[0] in ("read", "write")})
    place = {n: i for i, n in enumerate(places)}
    helpers = len(progs) - WARPS
    # steps taken by each | phases completed and arrivals of each barrier | places | states [helper][warp]
    start = ((0,) * len(progs), ((0, 0),) * len(names), (None,) * len(places), (None,) * (helpers * WARPS))
    seen, stack = {start}, [start]
    while stack:
        at, bars, held, states = stack.pop()
        moved = False
        for who, p in enumerate(progs):
            if at[who] == len(p):
                continue
            step, b, v, st = p[at[who]], bars, held, states
            if step[0] == "wait":
                if b[bar[step[1]]][0] % 2 == step[2]:  # the phase of that parity has not completed
                    continue
            elif step[0] == "arrive":
                done, n = b[bar[step[1]]]
                n += 1
                new = (done + 1, 0) if n == count[step[1]] else (done, n)
                b = b[: bar[step[1]]] + (new,) + b[bar[step[1]] + 1 :]
            elif step[0] == "read":
                if v[place[step[1]]] != step[2]:
                    return f"{step[1]} read for row {step[2]} holds row {v[place[step[1]]]}"
            elif step[0] == "write":
                v = v[: place[step[1]]] + (step[2],) + v[place[step[1]] + 1 :]
            elif step[0] == "state":
                k = step[1] * WARPS + who
                st = st[:k] + (step[2],) + st[k + 1 :]
            elif any(s != step[2] for s in st[step[1] * WARPS : (step[1] + 1) * WARPS]):
                return f"states merged for row {step[2]}: {st}"
            moved = True
            nxt = (at[:who] + (at[who] + 1,) + at[who + 1 :], b, v, st)
            if nxt not in seen:
                seen.add(nxt)
                stack.append(nxt)
        if not moved and any(a < len(p) for a, p in zip(at, progs)):
            return "everybody waits"
    return None


@pytest.mark.parametrize("name,lists,grad,helpers,lag", layouts())
def test_every_order_of_a_layout(name, lists, grad, helpers, lag):
    for late in {False, lag}:  # rows longer than the layout's limit run without lag
        assert faults(programs(grad, False, late, lists, helpers)) is None
    if grad and not lists:
        assert faults(programs(grad, True, False, lists, helpers)) is None  # from saved statistics


def test_the_model_finds_what_is_wrong():
    """One helper, the gradient one row behind, and nothing that holds the helper back."""
    assert faults(programs(True, False, True, False, 1)) is not None
    assert faults(programs(True, False, True, True, 1)) is None  # lists: it waits for `written`
