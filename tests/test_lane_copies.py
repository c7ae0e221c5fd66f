"""The compiler's register copies where lanes come together again.

Under high register pressure the compiler has placed copies of live registers (VGPR to
AGPR) between the label at which a divergent branch ends and the instruction that
switches its lanes on again: the lanes that were off keep what the target held, and a
thread number read back later is garbage. (A form of few_kernel at head dim 256 gave wrong
columns that way, with 472 registers; nothing in its source was wrong.) No test of
results finds it reliably, the listing does: every kernel is compiled to assembly and looked
through.
"""
import concurrent.futures as cf
import importlib.util
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "cron-root-attention_amd")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
COPY = re.compile(r"v_accvgpr_(write|read)_b32 \w+, [va]\d+|v_accvgpr_mov|v_mov_b(32|64)(_e32)? v\S+, v|scratch_"
                  r"|buffer_(store|load)\S+ .*\bs32\b")


def copies_before_lanes_return(asm):
    """(kernel, line, copies) of every place of an assembly listing."""
    found = []
    for m in re.finditer(r"^(_Z\w+):.*?\n(.*?)\n\s*\.section", asm, re.S | re.M):
        ends = set(re.findall(r"s_cbranch_execz (\.LBB\w+)", m[2]))
        copies = None  # since the label of such a block; None: not in one
        for n, line in enumerate(m[2].splitlines()):
            s = line.split(";")[0].strip()
            label = re.match(r"(\.LBB\w+):", s)
            if label:
                copies = [] if label[1] in ends else None
            elif copies is None or not s:
                continue
            elif s.startswith("s_or_b64 exec, exec"):
                if copies:
                    found.append((m[1], n, copies))
                copies = None
            elif s.startswith(("s_cbranch", "s_branch")) or (
                    re.search(r"\bexec\b", s) and not re.match(r"s_andn?2?_b64 vcc, exec", s)):
                copies = None
            elif COPY.match(s):
                copies.append(s)
    return found


SAMPLE = """_Z6kernelv:
	s_and_saveexec_b64 s[0:1], vcc
	s_cbranch_execz .LBB0_2
; %bb.1:
	v_mov_b32_e32 v1, v2
.LBB0_2:
{before}	s_or_b64 exec, exec, s[0:1]
{after}	s_endpgm
	.section	.rodata
"""


def test_what_is_looked_for():
    copy = "\tv_accvgpr_write_b32 a160, v56\n"
    fine = "\tv_writelane_b32 v255, s94, 29\n\ts_mov_b64 s[66:67], s[80:81]\n\tv_add_u32_e32 v3, 1, v4\n"
    (name, _, copies), = copies_before_lanes_return(SAMPLE.format(before=fine + copy, after=""))
    assert name == "_Z6kernelv" and copies == ["v_accvgpr_write_b32 a160, v56"]
    assert not copies_before_lanes_return(SAMPLE.format(before=fine, after=copy))


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
def test_no_kernel_copies_registers_with_lanes_off(tmp_path):
    spec = importlib.util.spec_from_file_location("cra_build", os.path.join(PKG, "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    csrc = os.path.join(PKG, "csrc")

    def listing(name):
        out = tmp_path / (name + ".s")
        subprocess.run([HIPCC, *build.common_flags(), "-S", "--cuda-device-only", os.path.join(csrc, name), "-o", str(out)],
                       check=True, capture_output=True, timeout=600)
        return out.read_text()
    sources = sorted(f for f in os.listdir(csrc) if f.endswith(".hip"))
    with cf.ThreadPoolExecutor(max_workers=8) as ex:
        texts = list(ex.map(listing, sources))
    assert sum(t.count("s_cbranch_execz") for t in texts) > 1000  # the listings are what they are taken for
    bad = {f: b for f, t in zip(sources, texts) if (b := copies_before_lanes_return(t))}
    assert not bad, bad
