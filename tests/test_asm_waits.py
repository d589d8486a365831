"""CPU: wait states that gfx950 leaves to the program, and m0, in the kernels as they
are built. The compiler keeps them for its own instructions and does not look into
inline assembly, where this library's loads into LDS are: a load needs 5 wait
states behind a vector instruction that writes the scalar registers of its
address, one into LDS another behind a write of m0. An instruction on the way
counts one, s_nop N counts N + 1; every way to a load is followed back, through
branches too."""
import functools
import pathlib
import re
import shutil
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
LIB = ROOT / "muse-glimmer-intel-serve_amd" / "libmgprims.so"
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"

LOADS = ("global_", "buffer_", "flat_", "scratch_")
# vector instructions whose second destination is in scalar registers
TWO = ("v_add_co", "v_addc_co", "v_sub_co", "v_subb_co", "v_subrev_co", "v_subbrev_co", "v_mad_u64", "v_mad_i64", "v_div_scale")
ENDS = ("s_branch", "s_endpgm", "s_setpc_b64")  # nothing falls through


@functools.lru_cache(None)
def scalars(text):
    """the scalar registers named in operands"""
    out = {"vcc"} if "vcc" in text else set()
    for a, b, one in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", text):
        out |= {int(one)} if one else set(range(int(a), int(b) + 1))
    return frozenset(out)


@functools.lru_cache(None)
def written(op, args):
    """the scalar registers that a vector instruction writes"""
    if not op.startswith("v_"):
        return frozenset()
    parts = re.split(r",\s*(?![^\[]*\])", args)
    return scalars(", ".join(parts[:2 if op.startswith(TWO) else 1]))


def parsed(lines):
    """[(op, operands, function)] of a disassembly with labels, and the branches to each label"""
    code, sources, name = [], {}, ""
    for line in lines:
        head = re.match(r"[0-9a-f]+ <(.*)>:", line)
        if head:
            label = re.fullmatch(r"L\d+", head[1])
            name = name if label else head[1]
            code.append(("label", head[1], name) if label else ("function", "", name))
        elif line[:1] in ("\t", " ") and line.strip():
            op, _, args = line.split("//")[0].strip().partition(" ")
            if op.startswith(("s_cbranch", "s_branch")):
                sources.setdefault((name, args.strip()), []).append(len(code))
            code.append((op, args.strip(), name))
    return code, sources


def wrote(code, sources, i, left, does):
    """whether an instruction for which `does` holds is on some way to the one at i, fewer than `left` wait states before"""
    todo, seen = [(i - 1, left)], {}
    while todo:
        j, n = todo.pop()
        if j < 0 or n <= 0 or seen.get(j, 0) >= n or code[j][0] == "function":
            continue
        seen[j] = n
        op, args, name = code[j]
        if op == "label":
            todo += [(k, n) for k in sources.get((name, args), ())]
            if code[j - 1][0] not in ENDS:
                todo.append((j - 1, n))
            continue
        if does(op, args):
            return True
        todo.append((j - 1, n - (int(args, 0) + 1 if op == "s_nop" else 1)))
    return False


def too_early(lines):
    """[(function, load, what it may read too early)], and how many loads into LDS there are"""
    code, sources = parsed(lines)
    bad, into_lds = [], 0
    for i, (op, args, name) in enumerate(code):
        if not op.startswith(LOADS):
            continue
        reads = scalars(args)
        if reads and wrote(code, sources, i, 5, lambda o, a: bool(written(o, a) & reads)):
            bad.append((name, f"{op} {args}", "address"))
        if "_lds_" in op:
            into_lds += 1
            if wrote(code, sources, i, 1, lambda o, a: o.startswith("s_") and a.startswith("m0")):
                bad.append((name, f"{op} {args}", "m0"))
    return bad, into_lds


@pytest.mark.parametrize("before,found", (
    ("v_readfirstlane_b32 s20, v1\ns_mov_b32 m0, s3\ns_nop 0", ["address"]),
    ("v_readfirstlane_b32 s21, v1\ns_mov_b32 m0, s3\ns_nop 2", ["address"]),
    ("v_readfirstlane_b32 s21, v1\ns_mov_b32 m0, s3\ns_nop 3", []),
    ("v_readfirstlane_b32 s22, v1\ns_mov_b32 m0, s3\ns_nop 0", []),
    ("v_cmp_gt_i64_e64 s[20:21], s[14:15], v[2:3]\ns_nop 0", ["address"]),
    ("v_mad_u64_u32 v[2:3], s[20:21], s3, v2, v[0:1]\ns_nop 0", ["address"]),
    ("v_add_u32_e32 v2, s20, v2\ns_mov_b32 m0, s3\ns_nop 0", []),
    ("s_nop 7\ns_mov_b32 m0, s3", ["m0"]),
    ("v_readlane_b32 s20, v1, 3\ns_branch L2\n<L1>\ns_nop 7\ns_branch L1\n<L2>\ns_nop 3", []),
    ("v_readlane_b32 s20, v1, 3\ns_branch L2\n<L1>\ns_nop 7\ns_branch L1\n<L2>\ns_nop 1", ["address"]),
    ("v_readlane_b32 s20, v1, 3\ns_branch L0\n<L1>\ns_nop 7\n<L0>\ns_nop 1", ["address"]),
    ("s_nop 7\n<L0>\ns_nop 0", ["address"])))  # (round the loop that the load ends)
def test_what_is_found(before, found):
    """the walk itself, on texts"""
    text = ["0000 <f>:"] + [f"0010 {x}:" if x.startswith("<") else f"\t{x}  // 00: 00" for x in before.split("\n")]
    text.append("\tglobal_load_lds_dwordx4 v0, s[20:21]  // 00: 00")
    text += ["\tv_readfirstlane_b32 s20, v7", "\ts_cbranch_scc1 L0", "\ts_endpgm"]
    bad, into_lds = too_early(text)
    assert [what for _, _, what in bad] == found and into_lds == 1


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    """the disassemblies of the device code that holds loads into LDS"""
    if not LIB.exists() or not shutil.which(OBJDUMP):
        pytest.skip("no library, or no disassembler, here")
    at = tmp_path_factory.mktemp("code")
    shutil.copy(LIB, at / "lib.so")  # (the device code is extracted beside it)
    subprocess.run([OBJDUMP, "--offloading", str(at / "lib.so")], check=True, capture_output=True)
    texts = [subprocess.run([OBJDUMP, "-d", "--symbolize-operands", str(o)], check=True, capture_output=True, text=True).stdout
             for o in sorted(at.glob("*gfx950"))]
    return [t.splitlines() for t in texts if "_load_lds_" in t]


def test_built_kernels(built):
    loads, bad = 0, []
    for lines in built:
        b, n = too_early(lines)
        bad += b
        loads += n
    assert loads > 1000  # (the labels and names are those that the walk reads)
    assert not bad, (len(bad), sorted({(f, what) for f, _, what in bad})[:12], bad[0])


def m0_misuse(lines):
    """uses of m0 beside a load's own: a scalar move into it, then s_nop, then the load into LDS that reads it"""
    code, _ = parsed(lines)
    for i, (op, args, name) in enumerate(code):
        if "_load_lds_" in op:
            if code[i - 1][0] != "s_nop" or code[i - 2][0] != "s_mov_b32" or not code[i - 2][1].startswith("m0"):
                yield name, op, args
        elif re.search(r"\bm0\b", args):
            if op != "s_mov_b32" or not args.startswith("m0") or not any("_load_lds_" in o for o, _, _ in code[i + 2:i + 3]):
                yield name, op, args


@pytest.mark.parametrize("text,found", (("s_mov_b32 m0, s1\ns_nop 3\nglobal_load_lds_dwordx4 v0, s[2:3]", 0),
                                        ("s_mov_b32 m0, s1\ns_nop 3\ns_nop 3\nglobal_load_lds_dwordx4 v0, s[2:3]", 2),
                                        ("s_mov_b32 m0, s1\ns_nop 3\nglobal_load_lds_dwordx4 v0, off\ns_mov_b32 s3, m0", 1),
                                        ("s_mov_b32 m0, s1\nv_movrels_b32_e32 v1, v2", 1)))
def test_what_is_found_of_m0(text, found):
    assert len(list(m0_misuse(["0000 <f>:"] + ["\t" + x for x in text.split("\n")]))) == found


def test_m0_is_the_loads_own(built):
    """The compiler cannot be told that inline assembly overwrites m0, and would not see it if it kept a value there: in
    kernels with such loads nothing else writes or reads it."""
    bad = []
    for lines in built:
        names = {name for op, _, name in parsed(lines)[0] if "_load_lds_" in op}
        bad += [m for m in m0_misuse(lines) if m[0] in names]
    assert not bad, (len(bad), bad[:4])
