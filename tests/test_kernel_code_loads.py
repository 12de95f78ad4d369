"""That the attention kernels' loads arrive: no register of a load is written over before it is read, on any way through the code, read from the
code objects that were built here.

The compiler did that to the loop of attention's parts for few rows, where the second halves of values loaded in pairs took part in the sums
as whatever was written into their registers meanwhile (arcinferzero_amd/csrc/kernels/attn_few.inc names the words for it).  A register of which a
load's others are read and it is not would be that again."""
import os
import re
import subprocess

import pytest

BUILD = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "arcinferzero_amd", "csrc", "build")
LLVM = "/opt/rocm/llvm/bin"
REGISTER = re.compile(r"(?<![\w\[])([va])(?:(\d+)\b|\[(\d+):(\d+)\])")
# instructions whose first operand is read, or is none of these registers
READS_ALL = re.compile(r"(global|buffer|ds|scratch|flat)_(store|write)|global_atomic|buffer_atomic|ds_(add|sub|max|min|or|and)_|v_cmp|v_readfirst|v_readlane|s_|buffer_load_\w+ .* lds")
READS_TOO = ("v_fmac", "v_pk_fmac", "v_dot", "v_mac", "v_writelane", "v_swap")


def registers(text):
    return {k + str(i) for k, a, b, c in REGISTER.findall(text) for i in (range(int(a), int(a) + 1) if a else range(int(b), int(c) + 1))}


def written_and_read(text):
    op, _, rest = text.partition(" ")
    if READS_ALL.match(text) and "rtn" not in op:
        return set(), registers(rest)
    first, _, others = rest.partition(",")
    w, r = registers(first), registers(others)
    if op.startswith(READS_TOO) or "_d16" in op or "dpp" in op or "sdwa" in op or "dst_sel" in rest:
        r |= w
    return w, r


def functions(code):
    """{name: [(text, the index that it may jump to)]}"""
    out, name = {}, None
    for line in code.splitlines():
        m = re.match(r"^([0-9a-f]+) <(\w+)>:", line)
        if m:
            name, start = m.group(2), int(m.group(1), 16)
            out[name] = []
            continue
        m = re.match(r"^\s+(\S.*?)\s*// ([0-9A-F]+): [0-9A-F ]+(?:<\w+\+0x([0-9a-f]+)>)?", line)
        if m and name:
            out[name].append((int(m.group(2), 16), m.group(1), None if m.group(3) is None else start + int(m.group(3), 16)))
    for n, ins in out.items():
        at = {a: i for i, (a, _, _) in enumerate(ins)}
        out[n] = [(t, at.get(to)) for _, t, to in ins]
    return out


def lost(ins):
    """The loads of memory of which some registers are read and others nowhere: [(text, those registers)]."""
    n = len(ins)
    steps = [written_and_read(t) for t, _ in ins]
    then = []
    for i, (t, to) in enumerate(ins):
        s = [to] if to is not None and t.startswith(("s_cbranch", "s_branch")) else []
        if not t.startswith(("s_branch", "s_endpgm", "s_setpc")) and i + 1 < n:
            s.append(i + 1)
        then.append(s)
    live, changed = [set() for _ in range(n)], True     # (in front of each)
    while changed:
        changed = False
        for i in range(n - 1, -1, -1):
            after = set().union(*(live[j] for j in then[i]))
            now = (after - steps[i][0]) | steps[i][1]
            if len(now) != len(live[i]):
                live[i], changed = now, True
    bad = []
    for i, (t, _) in enumerate(ins):
        if re.match(r"(global|buffer|flat)_load", t) and " lds" not in t:
            after = set().union(*(live[j] for j in then[i]))
            w = steps[i][0]
            if w - after:
                bad.append((t, sorted(w - after)))
    return bad


def test_what_is_looked_for():
    """The loop as the compiler had made it, and as it is to be."""
    def code(first):
        return [("global_load_dwordx2 v[86:87], v[70:71], off", None), ("s_waitcnt vmcnt(0)", None), (first, None), ("v_exp_f32_e32 v102, v99", None),
                ("v_xor_b32_e32 v86, 0x80808080, v86", None), ("v_xor_b32_e32 v88, 0x80808080, v87", None), ("v_add_f32_e32 v1, v86, v88", None),
                ("global_store_dword v[2:3], v1, off", None), ("s_cbranch_vccnz 65522", 0), ("s_endpgm", None)]
    assert lost(code("v_sub_f32_e32 v87, v102, v103")) == [("global_load_dwordx2 v[86:87], v[70:71], off", ["v87"])]
    assert lost(code("v_sub_f32_e32 v99, v102, v103")) == []


@pytest.mark.parametrize("module", ["attn_few", "attn_shared_few", "attn_many", "attn_shared", "kv", "rope", "norm_rope", "plan", "sample"])
def test_what_is_loaded_is_read(module, tmp_path):
    src, obj = os.path.join(BUILD, module + ".hsaco"), str(tmp_path / "o")
    if not os.path.exists(src) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("the code objects are not built here")
    subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", "--input=" + src, "--output=" + obj, "--unbundle"], check=True)
    code = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", obj], capture_output=True, text=True, check=True).stdout
    kernels = functions(code)
    assert sum(t.startswith("global_load") for ins in kernels.values() for t, _ in ins) > 3
    for name, ins in kernels.items():
        if ins:
            assert lost(ins) == [], name
