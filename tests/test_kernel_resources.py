"""No kernel of the product library spills to scratch (CPU: reads the built gfx950 code objects' metadata).

A scratch spill is a per-lane round trip through memory the roofline never counts (round 5: the bf16 loss kernel's
48 B/lane of spills were 25 MB of extra writes per C2 step). Every kernel the C1-C5 training steps launch must have
.private_segment_fixed_size == 0; the only kernels allowed scratch are the ones listed below, none of which any
benchmark configuration launches (every config runs hd = 16 or 64; hd 128 only through the generic fallback for
unaligned operands and the f32 mode at hd 128).
"""
import os
import re
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(REPO, "tools"))

ALLOWED = {
    # lane-per-query fallback kernels (unaligned operands / head dims without an MFMA kernel), hd 97-128
    r"attn_bwd_dkv_generic.*Li128E": "generic fallback at hd 128",
    # f32 (reference-precision) MFMA attention at hd 128: one wave per 32 queries holds a 32 x 128 f32 accumulator
    r"attn_(fwd|dq)_f32_kernel.*Li128E": "f32 mode at hd 128",
}
# kernels on the C1-C5 steps that must be present and spill-free (the round-5 offenders among them)
REQUIRED = [
    r"event_stream_kernelI14__hip_bfloat16",
    r"event_stream_kernelIf",
    r"attn_fwd_mfma_kernelILi64ELb1ELb0",
    r"attn_fwd_mfma_kernelILi16ELb1ELb0",
    r"attn_bwd_kernelILi64ELi2",
    r"gemm_bwd_pair_kernel",
    r"residual_ln_bwd_kernel",
    r"embed_joint_fwd_kernel",
]


def _kernels():
    build = os.path.join(REPO, "eventstreamgpt_amd", "csrc", "build")
    if not os.path.isdir(build) or not any(f.endswith(".o") for f in os.listdir(build)):
        pytest.skip("kernel objects not built (run __graft_entry__.build())")
    if not os.path.exists("/opt/rocm/lib/llvm/bin/llvm-objdump"):
        pytest.skip("ROCm LLVM tools absent")
    from kernel_resources import kernel_resources

    return kernel_resources(build)


def test_no_scratch_spills_in_product_kernels():
    ks = _kernels()
    assert len(ks) > 50
    bad = []
    for k in ks:
        if k.get("private_segment_fixed_size", 0) == 0:
            continue
        if any(re.search(p, k["name"]) for p in ALLOWED):
            continue
        bad.append((k["object"], k["private_segment_fixed_size"], k["name"]))
    assert not bad, "kernels spilling to scratch:\n" + "\n".join(map(str, bad))
    for pat in REQUIRED:
        hits = [k for k in ks if re.search(pat, k["name"])]
        assert hits, pat
        assert all(k.get("private_segment_fixed_size", 0) == 0 for k in hits), pat


def test_whole_form_of_the_shared_decode_attention_fits_its_plan():
    """Its plan counts on two waves a SIMD: one workgroup of eight waves a CU, or two of four. That is 256 registers (of both
    kinds) a lane at most."""
    ks = [k for k in _kernels() if "shared_whole_kernel" in k["name"]]
    assert len(ks) == 8
    assert [(k["name"], k["vgpr_count"]) for k in ks if k["vgpr_count"] > 256] == []


def test_dependency_graph_attention_backward_keeps_its_waves():
    """One query block per item, head size 64: the waves a SIMD that bound it, five up to six tokens (102 registers) and
    four up to eight (128), in both types."""
    seen = 0
    for k in _kernels():
        m = re.search(r"attn_bwd_small4I(?:f|14__hip_bfloat16)Li4ELi([468])ELb[01]ELi1ELb1E", k["name"])
        if m:
            seen += 1
            assert k["vgpr_count"] <= (128 if m.group(1) == "8" else 102), (k["name"], k["vgpr_count"])
    assert seen == 8
