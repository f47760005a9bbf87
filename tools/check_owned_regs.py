#!/usr/bin/env python3
"""Build-time audit of the kernels whose inline asm owns accumulator registers: fa_fwd_w64_kernel, its masked
forms (causal, ragged, both) and its key-split form, the fa_fwd_hd_kernel family and the fa_shared_prefix kernels.
In the latter, also the tables that a wave's lanes exchange through LDS at the start: see audit_exchange.

These kernels name a[..] literally in their instruction strings; the compiler does not know they hold
live values.  That is only sound while the compiler itself uses no accumulator register and spills
nothing in that kernel.  This script compiles the library's device code to assembly and fails if
any of them has scratch, spills, or any v_accvgpr_* / a[..] operand outside the #ASMSTART/#ASMEND
blocks, anywhere in the function (a kernel with early exits has several s_endpgm: the scan runs to the
function's end label).

    python tools/check_owned_regs.py [extra hipcc flags...]

Environment (experiment builds): FA_AUDIT_SRC = another source file, FA_AUDIT_KERNELS = comma-separated mangled
names to audit instead of the library's list, FA_AUDIT_KEEP = where to keep the assembly.
"""
import os
import re
import subprocess
import sys
import tempfile

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = os.path.join(ROOT, "flash-attention_amd", "csrc", "flash_attention_capi.hip")
KERNELS = ["_ZN2fa17fa_fwd_w64_kernelENS_9FwdParamsE", "_ZN2fa24fa_fwd_w64_causal_kernelENS_9FwdParamsE",
           "_ZN2fa24fa_fwd_w64_ragged_kernelENS_9FwdParamsE", "_ZN2fa31fa_fwd_w64_ragged_causal_kernelENS_9FwdParamsE",
           "_ZN2fa23fa_fwd_w64_split_kernelENS_9FwdParamsE", "_ZN2fa24fa_fwd_w64_varlen_kernelENS_9FwdParamsE", "_ZN2fa31fa_fwd_w64_varlen_causal_kernelENS_9FwdParamsE",
           "_ZN2fa16fa_fwd_hd_kernelILi256EEEvNS_9FwdParamsE",
           "_ZN2fa16fa_fwd_hd_kernelILi64EEEvNS_9FwdParamsE", "_ZN2fa23fa_fwd_hd_masked_kernelILi256EEEvNS_9FwdParamsE",
           "_ZN2fa23fa_fwd_hd_masked_kernelILi64EEEvNS_9FwdParamsE", "_ZN2fa23fa_fwd_hd_masked_kernelILi128EEEvNS_9FwdParamsE",
           "_ZN2fa22fa_fwd_hd_state_kernelILi64EEEvNS_9FwdParamsE", "_ZN2fa22fa_fwd_hd_state_kernelILi128EEEvNS_9FwdParamsE",
           "_ZN2fa22fa_fwd_hd_state_kernelILi256EEEvNS_9FwdParamsE"]

# the shared-prefix kernels: another translation unit, with its own flags (csrc/Makefile's PAGEDFLAGS)
PAGED_SRC = os.path.join(ROOT, "flash-attention_amd", "csrc", "flash_attention_paged.hip")
PAGED_FLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-mllvm", "-amdgpu-mfma-vgpr-form=1"]
PAGED_KERNELS = ["_ZN2fa%dfa_shared_prefix_%s_d%d_kernelENS_18SharedPrefixParamsE" % (len("fa_shared_prefix_%s_d%d_kernel" % (e, d)), e, d)
                 for e in ("f16", "bf16") for d in (64, 128, 256)]


def main():
    src = os.environ.get("FA_AUDIT_SRC", SRC)
    kernels = os.environ["FA_AUDIT_KERNELS"].split(",") if os.environ.get("FA_AUDIT_KERNELS") else KERNELS
    with tempfile.TemporaryDirectory() as tmp:
        out = os.path.join(tmp, "capi.s")
        cmd = ["/opt/rocm/bin/hipcc", "-O3", "-std=c++17", "--offload-arch=gfx950", "-fno-honor-nans", "-S",
               "--cuda-device-only", "-o", out, src] + sys.argv[1:]
        subprocess.run(cmd, check=True, stderr=subprocess.DEVNULL)
        text = open(out).read()
        if os.environ.get("FA_AUDIT_KEEP"):
            open(os.environ["FA_AUDIT_KEEP"], "w").write(text)
    for kernel in kernels:
        audit(text, kernel)
    if not os.environ.get("FA_AUDIT_KERNELS") and not sys.argv[1:]:
        with tempfile.TemporaryDirectory() as tmp:
            out = os.path.join(tmp, "paged.s")
            subprocess.run(["/opt/rocm/bin/hipcc", "-O3", "-std=c++17", "--offload-arch=gfx950"] + PAGED_FLAGS +
                           ["-S", "--cuda-device-only", "-o", out, PAGED_SRC], check=True, stderr=subprocess.DEVNULL)
            text = open(out).read()
        for kernel in PAGED_KERNELS:
            audit(text, kernel)
            audit_exchange(text, kernel)
    print("check_owned_regs: ok (no spills, no scratch, no compiler use of accumulator registers)")


def body_of(text, KERNEL):
    # the whole function body, up to its end label (a kernel with early exits has several s_endpgm)
    m = re.search(r"^" + KERNEL + r":.*?\n\.Lfunc_end\d+:", text, re.S | re.M)
    if not m:
        sys.exit("check_owned_regs: kernel not found in the assembly")
    return m


def audit_exchange(text, KERNEL):
    """Until the first barrier of the workgroup the lanes of a wave hand one another table entries through LDS: every LDS read
    there stands behind a wave barrier that stands behind the writes before it."""
    written = False
    for line in body_of(text, KERNEL).group(0).split("\n"):
        code = line.split(";")[0]
        if re.search(r"\bs_barrier\b", code):
            return
        if "wave barrier" in line:
            written = False
        elif re.search(r"\bds_write", code):
            written = True
        elif written and re.search(r"\bds_read", code):
            sys.exit("check_owned_regs: FAILED for " + KERNEL + "\n    an LDS read with no wave barrier behind the writes: " + code.strip())


def audit(text, KERNEL):
    m = body_of(text, KERNEL)
    problems = []
    in_asm = False
    for line in m.group(0).split("\n"):
        if "#ASMSTART" in line:
            in_asm = True
            continue
        if "#ASMEND" in line:
            in_asm = False
            continue
        code = line.split(";")[0]
        if not in_asm and (re.search(r"\bv_accvgpr", code) or re.search(r"\ba\[?\d", code)):
            problems.append("compiler-generated accumulator-register access: " + code.strip())
        if re.search(r"\bscratch_(load|store)", code):
            problems.append("scratch access: " + code.strip())
    meta = text[text.find(".amdhsa_kernel " + KERNEL):]
    meta = meta[:meta.find(".end_amdhsa_kernel")]
    for key in (".amdhsa_private_segment_fixed_size",):
        mm = re.search(key + r"\s+(\d+)", meta)
        if mm and int(mm.group(1)) != 0:
            problems.append(f"{key} = {mm.group(1)}")
    lanes = len(re.findall(r"\bv_(?:read|write)lane_b32", m.group(0)))
    if lanes:
        print(f"check_owned_regs: note: {KERNEL} keeps scalar values in vector lanes ({lanes} v_readlane/v_writelane)")
    if problems:
        print("check_owned_regs: FAILED for", KERNEL)
        for p in problems[:20]:
            print("   ", p)
        sys.exit(1)


if __name__ == "__main__":
    main()
