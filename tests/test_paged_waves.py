"""The paged decode's waves take part whole in its copies and matrix products (CPU only, needs hipcc).

A wave of paged_parts and paged_whole copies a chunk with all 64 lanes, whatever its lanes hold of lengths and page numbers: its branches
and loops have to be the wave's and not a lane's. A compiler that sees how a lane's value decides a vote can give some lanes a loop of their
own, and the others' copies then move half a chunk. This follows the execution mask through the compiled kernels, from the full wave that
a workgroup of whole waves starts with, and asks that it is full wherever a copy to LDS, a matrix instruction or a transposed read
stands.
"""
import os
import re
import subprocess

import pytest

from test_lds_dma_hazards import HIPCC, PKG

# A set of lanes: (path, whole). The path names parts of parts: () is all lanes, (7,) those that instruction 7 left of them,
# (-7,) the rest of that; whole: exactly those lanes, else some of them.
FULL = ((), True)


def _common(p, q):
    n = 0
    while n < min(len(p), len(q)) and p[n] == q[n]:
        n += 1
    return p[:n]


def _join(x, y):
    """What holds on either way."""
    return x if x == y else (_common(x[0], y[0]), False)


def _or(x, y):
    (p, e), (q, f) = x, y
    if f and p[:len(q)] == q:
        return y
    if e and q[:len(p)] == p:
        return x
    if e and f and p and q and p[:-1] == q[:-1] and p[-1] == -q[-1]:
        return p[:-1], True
    return _common(p, q), False


def _xor(x, y):
    (p, e), (q, f) = x, y
    if len(p) > len(q):
        (p, e), (q, f) = (q, f), (p, e)
    if e and f and len(q) == len(p) + 1 and q[:-1] == p:
        return p + (-q[-1],), True
    return _common(p, q), False


def _registers(text):
    regs = []
    for m in re.finditer(r"\b([sv])\[(\d+):(\d+)\]|\b([sv])(\d+)\b|\b(vcc|exec)\b", text):
        if m.group(1):
            regs += [f"{m.group(1)}{i}" for i in range(int(m.group(2)), int(m.group(3)) + 1)]
        elif m.group(4):
            regs.append(m.group(4) + m.group(5))
        else:
            regs += [m.group(6) + "0", m.group(6) + "1"]
    return regs


class _State(dict):
    """Registers' halves of sets of lanes: "s4" -> (set, 0 or 1); spilled ones under "v255:3"; what is not there is unknown."""

    def pair(self, text):
        if text.strip() == "-1":
            return FULL
        r = _registers(text)
        a, b = (self.get(r[0]), self.get(r[1])) if len(r) == 2 else (None, None)
        return a[0] if a and b and a[0] == b[0] and (a[1], b[1]) == (0, 1) else ((), False)

    def put(self, text, value):
        r = _registers(text)
        self[r[0]], self[r[1]] = (value, 0), (value, 1)

    def forget(self, regs):
        for r in regs:
            self.pop(r, None)
            if r[0] == "v" and r[1:].isdigit():
                for k in [k for k in self if k.startswith(r + ":")]:
                    del self[k]

    def renew(self, i):
        """Instruction i leaves other lanes than when it last ran."""
        for k, ((p, _), half) in list(self.items()):
            for n, a in enumerate(p):
                if abs(a) == i:
                    self[k] = ((p[:n], False), half)
                    break


def _step(i, op, args, st):
    """The state after instruction i (from 1 on)."""
    st = _State(st)
    if re.fullmatch(r"s_(and|andn2|or)_saveexec_b64", op):
        old, src = st.pair("exec"), st.pair(args[1])
        st.renew(i)
        old = (old[0], old[1]) if i not in map(abs, old[0]) else ((), False)
        if op == "s_or_saveexec_b64":
            new = _or(old, src)
        elif op == "s_andn2_saveexec_b64" and old[1] and src[1] and old[0] and src[0] and old[0][:-1] == src[0][:-1] and old[0][-1] == -src[0][-1]:
            new = src                                        # the other lanes of an if: none of the ones at hand
        elif op == "s_and_saveexec_b64" and old[1]:
            new = (old[0] + (i,), True)
        else:
            new = (old[0] if op == "s_and_saveexec_b64" else src[0], False)
        st.put(args[0], old)
        st.put("exec", new)
    elif op in ("s_or_b64", "s_xor_b64"):
        st.put(args[0], (_or if op == "s_or_b64" else _xor)(st.pair(args[1]), st.pair(args[2])))
    elif op in ("s_and_b64", "s_andn2_b64"):
        st.put(args[0], (st.pair(args[1])[0], False))
    elif op == "s_mov_b64":
        st.put(args[0], st.pair(args[1]))
    elif op == "s_mov_b32" and _registers(args[1]):
        v = st.get(_registers(args[1])[0])
        st.forget(_registers(args[0]))
        if v:
            st[_registers(args[0])[0]] = v
    elif op == "v_writelane_b32":
        v, at = st.get((_registers(args[1]) or [""])[0]), f"{args[0].strip()}:{args[2].strip()}"
        st.pop(at, None)
        if v:
            st[at] = v
    elif op == "v_readlane_b32":
        v = st.get(f"{args[1].strip()}:{args[2].strip()}")
        st.forget(_registers(args[0]))
        if v:
            st[args[0].strip()] = v
    elif args:
        carry = "_co_" in op or "div_scale" in op or op.startswith("v_mad_u64") or op.startswith("v_mad_i64")
        if op.startswith("v_cmpx"):
            st.put("exec", (st.pair("exec")[0], False))
        if not op.startswith(("s_cmp", "s_cbranch", "s_branch", "s_waitcnt", "s_bitcmp")):
            st.forget(_registers(args[0]) + (_registers(args[1]) if carry else []))
    return st


WHOLE = ("global_load_lds", "v_mfma", "ds_read_b64_tr")


def partial_instructions(lines):
    """(number of instructions looked at, those of them that not all lanes of a wave may run) of one kernel's assembly."""
    insts, labels = [], {}
    for raw in lines:
        s = raw.split(";")[0].strip()
        m = re.match(r"^([.\w$]+):", s)
        if m:
            labels[m.group(1)] = len(insts)
        elif s and not s.startswith("."):
            op, _, rest = s.partition(" ")
            op = re.sub(r"_e(32|64)$|_(sdwa|dpp)$", "", op.strip())
            insts.append((op, [a.strip() for a in re.split(r"[,\t]", rest.strip())] if rest.strip() else []))
    first = _State()
    first.put("exec", FULL)
    at, todo = {0: first}, [0]
    while todo:
        i = todo.pop()
        op, args = insts[i]
        st = _step(i + 1, op, args, at[i])
        if op == "s_endpgm":
            continue
        to = [] if op == "s_branch" else [i + 1]
        if op == "s_branch" or op.startswith("s_cbranch"):
            to.append(labels[args[-1]])
        assert not op.startswith(("s_setpc", "s_swappc", "s_call")), op
        for t in to:
            if t >= len(insts):
                continue
            if t not in at:
                at[t] = st
                todo.append(t)
                continue
            old, new = at[t], _State()
            for k in old.keys() & st.keys():
                if old[k][1] == st[k][1]:
                    new[k] = (_join(old[k][0], st[k][0]), old[k][1])
            if "exec0" not in new:
                new.put("exec", ((), False))
            if new != old:
                at[t] = new
                todo.append(t)
    seen = [i for i, (op, _) in enumerate(insts) if op.startswith(WHOLE) and i in at]
    return len(seen), [(i, insts[i][0]) for i in seen if at[i].pair("exec") != FULL]


def test_masks_are_followed():
    ok = """
        v_cmp_gt_i32_e32 vcc, s0, v0
        s_and_saveexec_b64 s[2:3], vcc
        s_cbranch_execz .L1
        v_mov_b32_e32 v1, 0
        .L1:
        s_or_b64 exec, exec, s[2:3]
        global_load_lds_dwordx4 v1, s[4:5]
        s_and_saveexec_b64 s[6:7], vcc
        s_xor_b64 s[6:7], exec, s[6:7]
        v_writelane_b32 v9, s6, 1
        v_writelane_b32 v9, s7, 2
        s_mov_b64 s[6:7], 0
        v_readlane_b32 s6, v9, 1
        v_readlane_b32 s7, v9, 2
        s_andn2_saveexec_b64 s[6:7], s[6:7]
        s_or_b64 exec, exec, s[6:7]
        v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], 0
        s_endpgm"""
    assert partial_instructions(ok.split("\n")) == (2, [])
    inside = ok.replace("v_mov_b32_e32 v1, 0", "global_load_lds_dwordx4 v1, s[4:5]")
    assert len(partial_instructions(inside.split("\n"))[1]) == 1
    lost = ok.replace("s_mov_b64 s[6:7], 0", "v_mov_b32_e32 v9, 0")
    assert len(partial_instructions(lost.split("\n"))[1]) == 1
    # lanes leave a loop one by one; the copy in it is theirs that are left, the one behind it everyone's
    loop = """
        s_mov_b64 s[2:3], 0
        .L1:
        global_load_lds_dwordx4 v1, s[4:5]
        v_cmp_gt_i32_e32 vcc, s0, v0
        s_or_b64 s[2:3], vcc, s[2:3]
        s_andn2_b64 exec, exec, s[2:3]
        s_cbranch_execnz .L1
        s_or_b64 exec, exec, s[2:3]
        s_endpgm"""
    assert partial_instructions(loop.split("\n"))[1] == [(1, "global_load_lds_dwordx4")]
    for whole in ("s_cbranch_vccnz .L1", "s_cbranch_scc1 .L1"):   # the wave's loop
        wave = re.sub(r"s_or_b64 s\[2:3\], vcc.*\n.*\n.*\n.*\n", whole + "\n", loop)
        assert partial_instructions(wave.split("\n")) == (1, [])


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_paged_decode_waves_stay_whole(tmp_path):
    # the Makefile's own line for this source, to assembly
    line = subprocess.run(["make", "-n", "-B", "_build/decode_paged.o"], cwd=PKG, capture_output=True, text=True, check=True).stdout
    line = [l for l in line.splitlines() if "decode_paged.hip" in l][0].split()
    out = tmp_path / "decode_paged.s"
    cmd = [HIPCC] + line[1:line.index("-c")] + ["--offload-device-only", "-S", "csrc/decode_paged.hip", "-o", str(out)]
    r = subprocess.run(cmd, cwd=PKG, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    text = out.read_text()
    names = re.findall(r"^(_ZN\S*paged_(?:parts|whole)\S*):", text, re.M)
    assert len(names) == 32 + 58                             # every instance of paged_parts, of paged_whole
    for name in names:
        body = re.search(rf"^{re.escape(name)}:.*?^\.Lfunc_end", text, re.M | re.S).group(0)
        count, bad = partial_instructions(body.split("\n"))
        assert count > 20 and not bad, f"{name}: {bad[:3]} of {count}"
    # and nothing spills to memory
    assert set(re.findall(r"\.amdhsa_private_segment_fixed_size (\d+)", text)) == {"0"}
