"""Instructions of the built library (p2pdl_amd/libp2pdl_hip.so).  No GPU needed.

No packed 32-bit float ones: some of their forms have given wrong results on this hardware now and then, with
no error, and the compiler makes them by itself from ordinary float code unless it is told not to (csrc/Makefile).
Of the scalar memory ones, loads only.
"""
import os
import re
import shutil
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(REPO, "tools"))
import isa_stats  # noqa: E402

SO = os.path.join(REPO, "p2pdl_amd", "libp2pdl_hip.so")


def test_no_packed_float_instructions():
    if not os.path.exists(os.path.join(isa_stats.LLVM, "llvm-objdump")) or shutil.which("true") is None:
        pytest.skip("ROCm LLVM tools not installed")
    funcs = isa_stats.functions(isa_stats.disassemble(SO))
    assert any("fedavg" in n for n in funcs) and any("robust" in n for n in funcs) and any("gemm_kernel" in n for n in funcs)
    packed = {n: sorted({op for op in ops if op.startswith("v_pk_") and "_f32" in op}) for n, ops in funcs.items()}
    assert not {n: ops for n, ops in packed.items() if ops}


def test_scalar_memory_instructions_are_loads():
    """Every scalar memory instruction is a load, the cache's invalidation or the clock: a list of what is allowed, so
    that one it does not know fails."""
    if not os.path.exists(os.path.join(isa_stats.LLVM, "llvm-objdump")) or shutil.which("true") is None:
        pytest.skip("ROCm LLVM tools not installed")
    allowed = re.compile(r"s_(buffer_)?load_(dword|dwordx2|dwordx4|dwordx8|dwordx16)|s_dcache_inv|s_memtime|s_memrealtime")
    memory = re.compile(r"s_.*(load|store|atomic|dcache|scratch|mem|probe)")
    found = {op for ops in isa_stats.functions(isa_stats.disassemble(SO)).values() for op in ops if memory.match(op)}
    assert any(op.startswith("s_load") for op in found)
    assert not {op for op in found if not allowed.fullmatch(op)}
