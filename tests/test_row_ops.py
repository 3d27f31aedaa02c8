"""The row operators without a GPU: refusals (every call is turned down before it reaches the GPU), the host's
view of strided rows, and what the built code of the large product looks like."""
import ctypes
import os
import re
import shutil
import subprocess
import sys

import pytest
import torch

from compression_amd import _lib, ops
from compression_amd._lib import MpcError


def test_rows_of_views():
    t = torch.zeros(4, 6, 8)
    assert ops._rows(t, "t") == (24, 8)
    assert ops._rows(t[:, :, :5], "t") == (24, 8)                       # a slice of wider rows
    assert ops._rows(t[::2, 0], "t") == (2, 96)
    assert ops._rows(t[:, :1, 1:4], "t") == (4, 48)                     # (the axis of one row has no say)
    assert ops._rows(t[0, 0], "t") == (1, 8)
    assert ops._rows(torch.zeros(8).expand(5, 8), "t") == (5, 0)        # a broadcast row
    assert ops._rows(torch.zeros(3, 7)[:, :1], "t") == (3, 7)
    assert ops._rows(torch.zeros(0, 7), "t") == (0, 7)
    for bad in (t[:, :4], t.transpose(0, 1)[..., :5]):
        with pytest.raises(MpcError, match="evenly spaced"):
            ops._rows(bad, "t")
    with pytest.raises(MpcError, match="consecutive"):
        ops._rows(t[..., ::2], "t")
    for bad in (torch.zeros(3, 0), torch.zeros(())):
        with pytest.raises(MpcError, match="at least one value"):
            ops._rows(bad, "t")


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    for call in (lambda: ops.rms_norm(x), lambda: ops.linear(x.half(), x.half()), lambda: ops.prior_balance(x),
                 lambda: ops.prior_balance_grad(x, x, x)):
        with pytest.raises(MpcError, match="no CPU path"):
            call()


def test_balance_takes_no_number_modulo_its_type():
    scores = torch.zeros(2, 8)
    assert ops._balance_args(scores, 1.0, 8, None)[7] == 8
    for top_k in (0, -1, 9, (1 << 32) + 1, 1 - (1 << 32)):
        with pytest.raises(MpcError, match="top_k"):
            ops._balance_args(scores, 1.0, top_k, None)
    with pytest.raises(MpcError, match="experts"):
        ops._balance_args(torch.zeros(1, 1).expand(2, (1 << 32) + 4), 1.0, 1, None)


def test_linear_workspace_of_a_bad_description_is_zero():
    lib = _lib.load()
    d = _lib.LinearDesc(_lib.MPC_TYPE_F32, _lib.MPC_TYPE_F32, 0, 4, 4, 4, 4, 4, 0, 4)
    assert lib.mpc_linear_workspace_bytes(ctypes.byref(d)) == 0
    assert lib.mpc_linear_workspace_bytes(None) == 0
    assert lib.mpc_prior_balance_workspace_bytes(-1, 64) == 0
    assert lib.mpc_prior_balance_workspace_bytes(16, 0) == 0
    assert lib.mpc_prior_balance_workspace_bytes(16, 1025) == 0
    assert lib.mpc_prior_balance_workspace_bytes(0, 64) > 0


def test_linear_refuses_strides_that_no_memory_has():
    lib = _lib.load()
    sizes = _lib.MPC_TYPE_BF16, _lib.MPC_TYPE_F32, 0, 64, 64, 1 << 16        # (a product whose K is split)
    assert lib.mpc_linear_workspace_bytes(ctypes.byref(_lib.LinearDesc(*sizes, 1 << 16, 1 << 16, 0, 64))) > 0
    for bad in ((1 << 61, 1 << 16, 0, 64), (1 << 16, 1 << 40, 0, 64), (1 << 16, 1 << 16, 1 << 62, 64), (1 << 16, 1 << 16, 0, 1 << 50)):
        assert lib.mpc_linear_workspace_bytes(ctypes.byref(_lib.LinearDesc(*sizes, *bad))) == 0


def test_entry_points_refuse_a_null_context():
    lib = _lib.load()
    d = _lib.LinearDesc(_lib.MPC_TYPE_F16, _lib.MPC_TYPE_F16, 0, 4, 4, 4, 4, 4, 0, 4)
    assert lib.mpc_linear_forward(None, ctypes.byref(d), None, None, None, None, None, None, None, 0, None) == -1
    assert lib.mpc_rms_norm(None, None, 0, None, 0, None, 1, 1, 0.0, 0, None, None, 0, None) == -1
    assert lib.mpc_prior_balance(None, None, 0, 1, 1, 1, 1, 1.0, 1, None, None, 0, None, None, None) == -1
    assert lib.mpc_prior_balance_grad(None, None, 0, 1, 1, 1, 1, 1.0, 1, None, None, None, None, None, 1, 1) == -1


# ---- the large product's matrix instructions, which the compiler does not see as such (inline asm) -------------------------
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LLVM = "/opt/rocm/lib/llvm/bin"


def _registers(text):
    out = set()
    for kind, lo, hi in re.findall(r"\b([va])\[(\d+):(\d+)\]", text):
        out |= {(kind, i) for i in range(int(lo), int(hi) + 1)}
    return out | {(kind, int(i)) for kind, i in re.findall(r"\b([va])(\d+)\b", text)}


@pytest.fixture(scope="module")
def big_kernels(tmp_path_factory):
    """{symbol: instructions} of linear_big_kernel in the built library."""
    lib = os.path.join(REPO, "compression_amd", "libmpc.so")
    if not os.path.exists(lib) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("needs the ROCm LLVM tools and a built libmpc.so")
    tmp = str(tmp_path_factory.mktemp("code"))
    copy = os.path.join(tmp, "lib.so")
    shutil.copy(lib, copy)
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", copy], cwd=tmp, check=True, capture_output=True)
    out = {}
    for name in sorted(os.listdir(tmp)):
        if "amdgcn" not in name:
            continue
        path = os.path.join(tmp, name)
        symbols = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--symbols", "--wide", path], capture_output=True, text=True, check=True).stdout
        for symbol in sorted(set(re.findall(r"\S*linear_big_kernel\S*", symbols))):
            if "." in symbol:                                  # (the descriptor, and notes about the kernel)
                continue
            text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", "--no-leading-addr",
                                   "--disassemble-symbols=" + symbol, path], capture_output=True, text=True, check=True).stdout
            lines = [re.sub(r"\s*//.*", "", x).strip() for x in text.split("\n")]
            out[symbol] = [x for x in lines if re.match(r"(v|s|ds|buffer|global|scratch)_\w+", x)]
    return out


def test_large_product_waits_for_its_matrix_instructions(big_kernels):
    """What the compiler would see to, had it known them: no vector instruction writes an operand within two instructions ahead of
    a matrix instruction that reads it, and none reads sums within 18 wait states of the last matrix instruction."""
    assert len(big_kernels) == 3
    for symbol, code in big_kernels.items():
        matrix = [i for i, x in enumerate(code) if x.startswith("v_mfma")]
        assert len(matrix) >= 128, symbol
        for i in matrix:
            used = _registers(code[i])
            for x in code[max(0, i - 2):i]:
                if x.startswith("v_") and not x.startswith(("v_mfma", "v_cmp", "v_readfirstlane")):
                    assert not _registers(x.split(None, 1)[1].split(",")[0]) & used, (symbol, x, code[i])
        waited = 0
        for x in code[matrix[-1] + 1:]:
            if waited >= 18:
                break
            if x.startswith("s_nop"):
                waited += int(x.split()[1]) + 1
            else:
                waited += 1
                assert not (x.startswith("v_") and any(kind == "a" for kind, _ in _registers(x))), (symbol, x)
        assert any(x.startswith("s_nop 15") for x in code[matrix[-1]:matrix[-1] + 12]), symbol


def test_large_product_keeps_its_sums_in_registers():
    sys.path.insert(0, os.path.join(REPO, "tools"))
    import kernel_registers
    if not os.path.exists(os.path.join(REPO, "compression_amd", "libmpc.so")) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("needs the ROCm LLVM tools and a built libmpc.so")
    big = {n: k for n, k in kernel_registers.kernels().items() if "linear_big_kernel" in n}
    assert len(big) == 3
    for name, k in big.items():
        assert k["agpr"] == 256 and k["vgpr"] + k["agpr"] <= 512 and k["scratch"] <= 64, (name, k)
