"""Checks a kernel's AMDGPU assembly for memory-to-LDS transfers that read a scalar register too soon after a vector
instruction wrote it.

The tiled products issue these transfers (global_load_lds_*, buffer_load_* with the lds modifier) as inline assembly, and the
compiler puts no wait states in front of instructions inside it.  A vector-memory instruction needs five between itself and a
vector instruction (v_readlane, v_readfirstlane, a compare) that wrote one of its scalar registers: a base that the compiler kept in a
lane would else be a stale one.  Dataflow over the control-flow graph: state = for each scalar register the wait states since
such a write, the fewest over all paths; every instruction is one, s_nop N is N + 1; a scalar instruction's write ends the watch.
"""
import functools
import re

import lds_wait_check as L

WAIT = 5
# a second scalar destination: carries and scale flags
CARRY = ("v_add_co", "v_addc_co", "v_sub_co", "v_subb_co", "v_subrev_co", "v_subbrev_co", "v_mad_u64_u32", "v_mad_i64_i32", "v_div_scale")


def _scalars(text):
    out = set()
    for m in re.finditer(r"\bs\[(\d+):(\d+)\]", text):
        out.update(range(int(m.group(1)), int(m.group(2)) + 1))
    for m in re.finditer(r"\bs(\d+)\b", text):
        out.add(int(m.group(1)))
    return out


@functools.lru_cache(maxsize=1 << 16)
def _effect(t):
    """Of instruction t: wait states, scalar registers that a transfer reads, that a scalar and that a vector instruction writes."""
    op = t.split()[0]
    parts = t[len(op):].split(",")
    reads = _scalars(t) if op.startswith(("global_", "buffer_")) and "lds" in t else ()
    by_scalar, by_vector = (), ()
    if op.startswith("s_") and not op.startswith(("s_nop", "s_waitcnt", "s_cmp", "s_bitcmp", "s_cbranch", "s_branch", "s_barrier")):
        by_scalar = _scalars(parts[0])
    if op.startswith("v_"):
        by_vector = _scalars(parts[0]) | (_scalars(parts[1]) if op.startswith(CARRY) and len(parts) > 1 else set())
    return int(parts[0], 0) + 1 if op == "s_nop" else 1, reads, by_scalar, by_vector


def _step(state, t):
    """(state after instruction t, scalar registers that it reads too soon)"""
    n, reads, by_scalar, by_vector = _effect(t)
    early = {r for r in reads if state.get(r, WAIT) < WAIT}
    new = {r: w + n for r, w in state.items() if w + n < WAIT} if state else {}
    for r in by_scalar:
        new.pop(r, None)
    for r in by_vector:
        new[r] = 0
    return new, early


def check_kernel(lines):
    """[(block, instruction, scalar registers)] for the lines of one kernel."""
    blocks, order = L._blocks(lines)
    state_in = {b: None for b in order}
    state_in["__entry"] = {}
    work, reports = ["__entry"], set()

    def flow(target, st):
        if target not in state_in:
            return
        old = state_in[target]
        new = dict(st) if old is None else {**old, **{r: min(w, old.get(r, WAIT)) for r, w in st.items()}}
        if old is None or new != old:
            state_in[target] = new
            work.append(target)

    while work:
        b = work.pop()
        st, live = state_in[b], True
        for t in blocks[b]:
            st, early = _step(st, t)
            if early:
                reports.add((b, t, tuple(sorted(early))))
            op = t.split()[0]
            if op.startswith("s_cbranch"):
                flow(t.split()[1], st)
            elif op == "s_branch":
                flow(t.split()[1], st)
                live = False
                break
            elif op in ("s_endpgm", "s_setpc_b64"):
                live = False
                break
        i = order.index(b)
        if live and i + 1 < len(order):
            flow(order[i + 1], st)
    return sorted(reports)


def check(path):
    """({kernel: findings}, number of transfers) over all kernels of an assembly file."""
    src = open(path).read().splitlines()
    # a kernel: from its symbol's label to its descriptor
    found, transfers, start, name = {}, 0, None, None
    kinds = {m.group(1) for ln in src for m in [re.match(r"\s*\.amdhsa_kernel\s+(\S+)", ln)] if m}
    for i, ln in enumerate(src):
        m = re.match(r"^([A-Za-z_]\S*):", ln)
        if m and m.group(1) in kinds:
            start, name = i, m.group(1)
        if start is not None and ".amdhsa_kernel" in ln:
            body = src[start + 1:i]
            transfers += sum(1 for t in body if re.match(r"\s+(global|buffer)_load", t) and "lds" in t.split(";")[0])
            found[name] = check_kernel(body)
            start = None
    return {k: v for k, v in found.items() if v}, transfers
