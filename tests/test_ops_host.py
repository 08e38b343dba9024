"""libdgnn_ops.so on the CPU: what it exports, the argument blocks the Python mirror packs, and every refusal of the C ABI.  Nothing is
launched here: a call that passes its checks is given a device that does not exist."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT
from test_cabi_host import _declared_symbols, _exported

NO_DEVICE = 1 << 20
OK, HIP_ERROR, BAD_ARGUMENT, UNSUPPORTED = 0, -3, -4, -6
F16, BF16, F32, I32, I64 = range(5)


@pytest.fixture(scope="module")
def ops(api):
    from dream_go_amd import ops as module
    return module


def test_the_library_exports_its_header_and_nothing_else(ops):
    assert _exported(ops.OPS_LIB_PATH) == _declared_symbols("dgnn_ops.h") == sorted(name for name, _, _ in ops.SYMBOLS)


def test_the_argument_blocks_are_the_headers_structs(ops, tmp_path):
    fields = {"dgnn_dense_args": (ops._DENSE, "activation"), "dgnn_group_norm_args": (ops._GROUP_NORM, "activation"),
              "dgnn_logits_args": (ops._LOGITS, "history_type")}
    lines = "".join(f'printf("%zu %zu\\n", sizeof({n}), offsetof({n}, {last}));' for n, (_, last) in fields.items())
    (tmp_path / "s.c").write_text(f'#include "dgnn_ops.h"\n#include <stdio.h>\nint main(void) {{ {lines} return 0; }}\n')
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "s"), str(tmp_path / "s.c")], check=True)
    out = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()
    for i, (block, _) in enumerate(fields.values()):
        assert block.size == int(out[2 * i])
        assert np.frombuffer(block.pack(*([0] * (len(block.unpack(bytes(block.size))) - 1)), 77), dtype=np.int32)[int(out[2 * i + 1]) // 4] == 77


DENSE = dict(x=0x10000, w=0x20000, bias=0x30000, z=0x40000, y=0x50000, workspace=0x100000, workspace_bytes=1 << 40, m=4, n=8, k=16, ldx=16, ldw=16, ldz=8, ldy=8, alpha1=1.0, alpha2=1.0,
             type=F16, out_type=F16, bias_type=F16, activation=0)
GROUP_NORM = dict(x=0x10000, weight=0x20000, bias=0x30000, z=0x40000, y=0x50000, workspace=0x100000, workspace_bytes=1 << 40, n=2, p=5, c=16,
                  groups=4, x_n=80, x_p=16, z_n=80, z_p=16, y_n=80, y_p=16, eps=1e-5, type=F16, affine_type=F32, activation=4)
LOGITS = dict(logits=0x10000, out=0x20000, mask=0x30000, bias=0x40000, history=0x50000, lengths=0x60000, prompt_lengths=0x70000, repetition=0,
              presence=0x80000, frequency=0x90000, b=3, v=100, t=7, ld_logits=100, ld_out=100, ld_mask=4, ld_bias=0, ld_history=7,
              repetition_all=1.0, presence_all=0.0, frequency_all=0.0, type=F16, out_type=F32, bias_type=F32, history_type=I32)


def call(ops, base, device=NO_DEVICE, **changes):
    block, fn = {id(DENSE): (ops._DENSE, ops.lib.dgnn_dense), id(GROUP_NORM): (ops._GROUP_NORM, ops.lib.dgnn_group_norm),
                 id(LOGITS): (ops._LOGITS, ops.lib.dgnn_adjust_logits)}[id(base)]
    assert set(changes) <= set(base)
    return fn(device, None, block.pack(*{**base, **changes}.values()))


@pytest.mark.parametrize("base,changes", [
    (DENSE, {}), (DENSE, dict(z=0)), (DENSE, dict(bias=0)), (DENSE, dict(ldz=0)), (DENSE, dict(k=0, x=0, w=0)), (DENSE, dict(ldx=0)),
    (DENSE, dict(z=0x50000)), (DENSE, dict(out_type=F32)), (DENSE, dict(type=BF16, out_type=BF16, bias_type=F32)),
    (DENSE, dict(x=0x10002, ldx=17, m=1, ldy=0)),
    (DENSE, dict(x=0x50000 + 16, ldx=32, ldy=32)),                       # x and y are columns of one buffer
    (GROUP_NORM, {}), (GROUP_NORM, dict(y=0x10000)), (GROUP_NORM, dict(y=0x40000)), (GROUP_NORM, dict(weight=0, bias=0, z=0)),
    (GROUP_NORM, dict(eps=0.0)), (GROUP_NORM, dict(x_n=0)), (GROUP_NORM, dict(z_n=0, z_p=0)), (GROUP_NORM, dict(groups=16)),
    (GROUP_NORM, dict(x=0x50000 + 32, x_p=64, x_n=320, y_p=64, y_n=320)),
    (LOGITS, {}), (LOGITS, dict(mask=0, bias=0, history=0)), (LOGITS, dict(out=0x10000, out_type=F16)), (LOGITS, dict(ld_mask=0)),
    (LOGITS, dict(history_type=I64)), (LOGITS, dict(repetition=0xa0000, repetition_all=-1.0)),
])
def test_what_is_allowed_gets_as_far_as_the_device(ops, base, changes):
    assert call(ops, base, **changes) == HIP_ERROR
    assert ops.lib.dgnn_ops_last_hip_error() != 0
    assert call(ops, base, device=-1, **changes) == BAD_ARGUMENT


@pytest.mark.parametrize("base,changes", [
    (DENSE, dict(m=0)), (DENSE, dict(n=0)), (DENSE, dict(m=0, x=0, y=0, z=0)),
    (GROUP_NORM, dict(n=0)), (GROUP_NORM, dict(p=0)), (GROUP_NORM, dict(c=0, groups=1)),
    (LOGITS, dict(b=0)), (LOGITS, dict(v=0)),
])
def test_nothing_to_do_is_done(ops, base, changes):
    assert call(ops, base, **changes) == OK


@pytest.mark.parametrize("base,changes,status", [
    (DENSE, dict(x=0), BAD_ARGUMENT), (DENSE, dict(w=0), BAD_ARGUMENT), (DENSE, dict(y=0), BAD_ARGUMENT),
    (DENSE, dict(m=-1), BAD_ARGUMENT), (DENSE, dict(n=1 << 31), BAD_ARGUMENT), (DENSE, dict(k=1 << 31), BAD_ARGUMENT),
    (DENSE, dict(ldy=7), BAD_ARGUMENT), (DENSE, dict(ldy=0), BAD_ARGUMENT), (DENSE, dict(ldx=-16), BAD_ARGUMENT), (DENSE, dict(ldw=1 << 60), BAD_ARGUMENT),
    (DENSE, dict(x=0x10001), BAD_ARGUMENT), (DENSE, dict(y=0x50002, out_type=F32), BAD_ARGUMENT), (DENSE, dict(bias=0x30002, bias_type=F32), BAD_ARGUMENT),
    (DENSE, dict(y=0x10000), BAD_ARGUMENT), (DENSE, dict(y=0x20010), BAD_ARGUMENT), (DENSE, dict(z=0x50002), BAD_ARGUMENT), (DENSE, dict(z=0x50000, ldz=0), BAD_ARGUMENT),
    (DENSE, dict(bias=0x50000), BAD_ARGUMENT),
    (DENSE, dict(x=0x50000 + 14, ldx=32, ldy=32), BAD_ARGUMENT),         # columns of one buffer that meet
    (DENSE, dict(activation=5), BAD_ARGUMENT), (DENSE, dict(activation=-1), BAD_ARGUMENT), (DENSE, dict(type=7), BAD_ARGUMENT),
    (DENSE, dict(type=F32, out_type=F32, bias_type=F32), UNSUPPORTED), (DENSE, dict(out_type=BF16), UNSUPPORTED), (DENSE, dict(bias_type=BF16), UNSUPPORTED),
    (GROUP_NORM, dict(x=0), BAD_ARGUMENT), (GROUP_NORM, dict(y=0), BAD_ARGUMENT), (GROUP_NORM, dict(groups=0), BAD_ARGUMENT),
    (GROUP_NORM, dict(groups=3), BAD_ARGUMENT), (GROUP_NORM, dict(groups=32), BAD_ARGUMENT), (GROUP_NORM, dict(eps=-1e-5), BAD_ARGUMENT),
    (GROUP_NORM, dict(eps=float("nan")), BAD_ARGUMENT), (GROUP_NORM, dict(eps=float("inf")), BAD_ARGUMENT), (GROUP_NORM, dict(y_p=15), BAD_ARGUMENT),
    (GROUP_NORM, dict(y_n=79), BAD_ARGUMENT), (GROUP_NORM, dict(y_n=0), BAD_ARGUMENT), (GROUP_NORM, dict(x_p=-16), BAD_ARGUMENT),
    (GROUP_NORM, dict(y=0x10020), BAD_ARGUMENT), (GROUP_NORM, dict(y=0x10000, y_p=32, y_n=160), BAD_ARGUMENT), (GROUP_NORM, dict(y=0x40002), BAD_ARGUMENT),
    (GROUP_NORM, dict(weight=0x50000), BAD_ARGUMENT), (GROUP_NORM, dict(affine_type=BF16), UNSUPPORTED), (GROUP_NORM, dict(type=9), BAD_ARGUMENT),
    (GROUP_NORM, dict(activation=9), BAD_ARGUMENT), (GROUP_NORM, dict(x=0x10001), BAD_ARGUMENT), (GROUP_NORM, dict(weight=0x20002), BAD_ARGUMENT),
    (LOGITS, dict(logits=0), BAD_ARGUMENT), (LOGITS, dict(out=0), BAD_ARGUMENT), (LOGITS, dict(ld_out=99), BAD_ARGUMENT), (LOGITS, dict(t=-1), BAD_ARGUMENT),
    (LOGITS, dict(v=1 << 31), BAD_ARGUMENT), (LOGITS, dict(repetition_all=0.0), BAD_ARGUMENT), (LOGITS, dict(repetition_all=float("nan")), BAD_ARGUMENT),
    (LOGITS, dict(presence=0, presence_all=float("inf")), BAD_ARGUMENT), (LOGITS, dict(frequency=0, frequency_all=float("nan")), BAD_ARGUMENT),
    (LOGITS, dict(out=0x10000), BAD_ARGUMENT), (LOGITS, dict(out=0x10064, out_type=F16), BAD_ARGUMENT), (LOGITS, dict(mask=0x30001), BAD_ARGUMENT),
    (LOGITS, dict(history=0x50004, history_type=I64), BAD_ARGUMENT), (LOGITS, dict(history_type=F32), BAD_ARGUMENT), (LOGITS, dict(lengths=0x60002), BAD_ARGUMENT),
    (LOGITS, dict(bias_type=BF16), UNSUPPORTED), (LOGITS, dict(out_type=BF16), UNSUPPORTED), (LOGITS, dict(type=I32), BAD_ARGUMENT),
    (LOGITS, dict(mask=0x20010), BAD_ARGUMENT), (LOGITS, dict(bias=0x20000), BAD_ARGUMENT), (LOGITS, dict(history=0x20000), BAD_ARGUMENT),
    (LOGITS, dict(frequency=0x20000), BAD_ARGUMENT), (LOGITS, dict(ld_history=-1), BAD_ARGUMENT),
])
def test_refusals(ops, base, changes, status):
    assert call(ops, base, **changes) == status


def test_null_argument_blocks(ops):
    need = ctypes.c_int64(5)
    assert ops.lib.dgnn_dense_workspace(None, need) == BAD_ARGUMENT and need.value == 0
    assert ops.lib.dgnn_dense_workspace(ops._DENSE.pack(*DENSE.values()), None) == BAD_ARGUMENT
    for fn in (ops.lib.dgnn_dense, ops.lib.dgnn_group_norm, ops.lib.dgnn_adjust_logits):
        assert fn(0, None, None) == BAD_ARGUMENT
    assert ops.lib.dgnn_group_norm_workspace(None, need) == BAD_ARGUMENT and need.value == 0
    assert ops.lib.dgnn_group_norm_workspace(ops._GROUP_NORM.pack(*GROUP_NORM.values()), None) == BAD_ARGUMENT


@pytest.mark.parametrize("shape", [(1, 361, 64, 8), (256, 361, 256, 32), (1, 1 << 18, 320, 32), (8, 1 << 14, 320, 32), (1, 1, 4096, 1), (1, 1 << 20, 3, 3)])
def test_a_workspace_that_is_too_small_is_refused(ops, shape):
    n, p, c, groups = shape
    args = dict(GROUP_NORM, n=n, p=p, c=c, groups=groups, x_n=p * c, x_p=c, y_n=p * c, y_p=c, z=0, x=1 << 40, y=1 << 42)
    need = ctypes.c_int64()
    assert ops.lib.dgnn_group_norm_workspace(ops._GROUP_NORM.pack(*args.values()), need) == OK
    assert 0 <= need.value < 1 << 28
    if need.value:
        for bad in (dict(workspace=0), dict(workspace_bytes=need.value - 1), dict(workspace=0x100080)):
            assert ops.lib.dgnn_group_norm(NO_DEVICE, None, ops._GROUP_NORM.pack(*{**args, **bad}.values())) == BAD_ARGUMENT
    assert ops.lib.dgnn_group_norm(NO_DEVICE, None, ops._GROUP_NORM.pack(*{**args, "workspace_bytes": need.value}.values())) == HIP_ERROR


@pytest.mark.parametrize("m,n,k,first,pad", [(1, 362, 2888, 0, 0), (16, 512, 8192, 0, 0), (1000, 1000, 1001, 0, 0), (300, 300, 320, 2, 0), (4096, 4096, 4095, 0, 1),
                                             (8192, 4096, 16384, 0, 0), (64, 64, 1 << 20, 0, 0), (1 << 20, 8, 64, 0, 0), (20, 20, (1 << 31) - 1, 0, 0)])
def test_the_workspace_of_a_dense_layer(ops, m, n, k, first, pad):
    args = dict(DENSE, x=(1 << 44) + first, w=1 << 45, y=1 << 46, z=0, m=m, n=n, k=k, ldx=k + pad, ldw=k, ldy=n)
    need = ctypes.c_int64()
    assert ops.lib.dgnn_dense_workspace(ops._DENSE.pack(*args.values()), need) == OK
    # never more than a copy of both operands, rows rounded up, and sixteen times the outputs in fp32
    assert 0 <= need.value <= 2 * (m + n) * (k + 64) + 64 * m * n + 1024
    if need.value:
        for bad in (dict(workspace=0), dict(workspace_bytes=need.value - 1), dict(workspace=0x100080)):
            assert ops.lib.dgnn_dense(NO_DEVICE, None, ops._DENSE.pack(*{**args, **bad}.values())) == BAD_ARGUMENT
    assert ops.lib.dgnn_dense(NO_DEVICE, None, ops._DENSE.pack(*{**args, "workspace_bytes": need.value}.values())) == HIP_ERROR


def test_tensors_of_the_cpu_are_refused(ops, api):
    import torch
    x = torch.zeros(4, 16, dtype=torch.float16)
    for run in (lambda: ops.dense(x, x), lambda: ops.group_norm(x, 4), lambda: ops.adjust_logits(x), lambda: ops.dense(x.numpy(), x)):
        with pytest.raises(api.Error) as e:
            run()
        assert e.value.status == api.BAD_ARGUMENT


@pytest.mark.parametrize("n", [1, 512])
@pytest.mark.parametrize("p,c,lanes,type_", [((1 << 31) - 1, 8, 1, F16), (1 << 28, 64, 8, BF16), ((1 << 29) - 64, 256, 64, F32), (1 << 20, 320, None, F16)])
def test_no_thread_adds_up_more_rows_than_the_sums_are_good_for(ops, n, p, c, lanes, type_):
    """A workspace holds eight bytes for every share of the positions; a share's rows are dealt to 512 threads, `lanes` of them side by side."""
    args = dict(GROUP_NORM, n=n, p=p, c=c, groups=1 if lanes else 32, x_n=p * c, x_p=c, y_n=p * c, y_p=c, z=0, x=1 << 50, y=1 << 54, type=type_, affine_type=F32)
    need = ctypes.c_int64()
    assert ops.lib.dgnn_group_norm_workspace(ops._GROUP_NORM.pack(*args.values()), need) == OK
    shares = need.value // (8 * n * args["groups"])
    assert 0 < shares <= 65535                                                # a grid's second extent
    assert -(-p // shares) <= 2048 * (512 // (lanes or 64 // 4))


def test_channels_are_counted_without_overflow(tmp_path):
    """Up to 2^31 - 1 channels.  An overflow is no constant expression: the compiler refuses it."""
    cases = [(0, 8, 8, 0), (0, 8, 5, 3), (8, 8, 13, 3), (8, 8, 16, 0), (0, 4, 1, 3), (2147483640, 8, 2147483647, 1), (2147483640, 8, 2147483646, 2),
             (2147483632, 8, 2147483647, 0), (2147483646, 1, 2147483647, 0), (2147483644, 4, 2147483647, 1)]
    lines = "".join(f"static_assert(dgnn::ops::overhang({c}, {width}, {channels}) == {want});\n" for c, width, channels, want in cases)
    (tmp_path / "s.cpp").write_text('#include "ops.h"\n' + lines)
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I", os.path.join(ROOT, "dream-go_amd", "csrc"), "-fsyntax-only", str(tmp_path / "s.cpp")],
                   check=True)


def test_what_carries_gradients_is_seen(ops):
    import torch
    import torch.autograd.forward_ad as forward
    x, leaf = torch.ones(3), torch.ones(3, requires_grad=True)
    assert ops._records(x, None, leaf) and not ops._records(x, None)
    with torch.no_grad():
        assert not ops._records(leaf)
    with forward.dual_level():
        dual = forward.make_dual(x, torch.ones(3))
        assert ops._records(None, dual) and not ops._records(x, None)
        with torch.no_grad():
            assert ops._records(x, dual) and not ops._records(leaf, forward.unpack_dual(dual).primal)
    assert not ops._records(x)


def test_numbers(ops, api):
    import torch
    learned = torch.tensor(0.5, requires_grad=True)
    for bad in (None, "1", b"1", 1j, [1.0], {}, 1 << 2000, torch.ones(2), learned):
        with pytest.raises(api.Error) as e:
            ops._number("dense", "alpha1", bad)
        assert e.value.status == (api.UNSUPPORTED if bad is learned else api.BAD_ARGUMENT) and str(e.value).count("dense")
    for good in (0, 2, True, 0.5, np.float32(0.5), np.int64(3), torch.tensor(0.5), learned.detach()):
        assert ops._number("dense", "alpha1", good) == float(good)
    with torch.no_grad():
        assert ops._number("dense", "alpha1", learned) == 0.5
    with pytest.raises(api.Error) as e:
        ops._launch("group_norm", None, None, 0, ops._GROUP_NORM, [0] * 11 + [1 << 70] + [0] * 6 + [1.0] + [0] * 3)
    assert e.value.status == api.BAD_ARGUMENT
