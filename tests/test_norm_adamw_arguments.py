"""What the norm behind a fold, its backward, and the AdamW plan refuse, and how a call is laid out.  No GPU: refused
calls and plans never touch a device."""
import ctypes
import os
import subprocess

import pytest

import megray_amd as mr

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AR, RS = mr.Collective.ALL_REDUCE, mr.Collective.REDUCE_SCATTER
BF16, F16, F32, E4M3, I8 = mr.DType.BFLOAT16, mr.DType.FLOAT16, mr.DType.FLOAT32, mr.DType.FLOAT8_E4M3, mr.DType.INT8
MIB = 1 << 20


def buffers(count, first=1):
    """Addresses far apart that nothing ever reads."""
    return [(first + i) * 64 * MIB for i in range(count)]


def forward(collective=AR, n=2, rows=4, cols=64, dtype=BF16, eps=1e-5, **changed):
    args = dict(sendbuffs=buffers(n), outs=buffers(n, 40), weight=100 * 64 * MIB, residuals=buffers(1 if collective == AR else n, 80),
                residual_outs=buffers(n, 120))
    args.update(changed)
    return mr.RmsNormPlan(collective, args.pop("sendbuffs"), args.pop("outs"), args.pop("weight"), rows, cols, dtype, eps, **args)


def backward(collective=AR, n=2, rows=4, cols=64, dtype=BF16, eps=1e-5, **changed):
    args = dict(sendbuffs=buffers(n), hiddens=buffers(1 if collective == AR else n, 40), weight=100 * 64 * MIB,
                residual_out_grads=buffers(n, 120), weight_grads=buffers(n, 160), workspace=200 * 64 * MIB, workspace_bytes=32 * MIB)
    args.update(changed)
    return mr.RmsNormBackwardPlan(collective, args.pop("sendbuffs"), args.pop("hiddens"), args.pop("weight"),
                                  args.pop("residual_out_grads"), rows, cols, dtype, eps, **args)


def refused(make, match, **changed):
    with pytest.raises(mr.MegRayError, match=match) as e:
        make(**changed)
    assert e.value.status == mr.Status.INVALID_ARGUMENT


@pytest.mark.parametrize("collective", [AR, RS])
def test_calls_that_are_allowed(collective):
    assert forward(collective).launch_count == 1
    assert forward(collective, residuals=None, residual_outs=None).launch_count == 1
    assert forward(collective, rows=0).launch_count == 0
    assert forward(collective, out_dtype=E4M3, scales=buffers(2, 180)).launch_count == 1
    assert forward(collective, dtype=F16, residual_dtype=F32, weight_dtype=F32).launch_count == 1
    for cols in (1, 7, 8, 9, 511, 513, 1025, 2049, 4097, 8193, 16385, 40000):
        assert forward(collective, cols=cols).launch_count == 1
        assert backward(collective, cols=cols, rows=2).launch_count == 2
    assert backward(collective).launch_count == 2
    assert backward(collective, weight_grads=None, workspace=None, workspace_bytes=0).launch_count == 1
    assert backward(collective, residual_out_grads=None).launch_count == 2
    assert backward(collective, rows=0).launch_count == 1  # the weight gradients are zero then
    assert backward(collective, send_grads=buffers(2, 220), residual_grads=buffers(1 if collective == AR else 2, 240),
                    residual_dtype=F32).launch_count == 2


def test_in_place_calls():
    n, rows, cols = 3, 4, 64
    send = buffers(n)
    forward(n=n, outs=send)
    forward(n=n, residual_outs=buffers(1, 80) + buffers(2, 120))  # one rank's copy of the residual is the one that is read
    own = [b + r * rows * cols * 2 for r, b in enumerate(send)]
    forward(RS, n=n, rows=rows, outs=own, residuals=buffers(n, 80), residual_outs=buffers(n, 80))
    refused(forward, "out of place", collective=RS, n=n, rows=rows, outs=send)
    refused(forward, "out of place", n=n, outs=[b + 2 for b in send])
    refused(forward, "out of place", n=n, outs=send[1:] + send[:1])
    refused(forward, "out of place", n=n, outs=send, out_stride=72)
    refused(forward, "out of place", n=n, outs=send, out_dtype=E4M3, scales=buffers(n, 180))
    refused(forward, "out of place", n=n, residual_outs=send)
    backward(n=n, send_grads=send)
    backward(n=n, residual_out_grads=buffers(1, 40) + buffers(2, 120))
    backward(RS, n=n, send_grads=own, residual_grads=buffers(n, 240), residual_out_grads=buffers(n, 240))
    refused(backward, "out of place", collective=RS, n=n, send_grads=send)


def test_columns_of_one_matrix_are_apart():
    """Outputs and inputs that interleave row by row, the column ranges of one wider matrix, do not overlap."""
    base = 64 * MIB
    forward(n=1, cols=64, sendbuffs=[base], outs=[base + 128], send_stride=128, out_stride=128)
    forward(n=1, cols=64, sendbuffs=[base + 128], outs=[base], send_stride=128, out_stride=128)
    refused(forward, "out of place", n=1, cols=64, sendbuffs=[base], outs=[base + 126], send_stride=128, out_stride=128)
    refused(forward, "out of place", n=1, cols=64, sendbuffs=[base], outs=[base + 130], send_stride=128, out_stride=128)
    refused(forward, "out of place", n=1, cols=64, sendbuffs=[base], outs=[base + 128], send_stride=128, out_stride=120)


@pytest.mark.parametrize("make", [forward, backward])
def test_what_both_directions_refuse(make):
    refused(make, "all_reduce or a reduce_scatter", collective=mr.Collective.ALL_GATHER)
    refused(make, "unknown dtype", dtype=mr.DType.FLOAT64)
    refused(make, "unknown dtype", dtype=E4M3)
    refused(make, "unknown residual dtype", residual_dtype=I8)
    refused(make, "the residual's dtype", dtype=F16, residual_dtype=BF16)
    refused(make, "the weight's dtype", dtype=F32, weight_dtype=F16)
    refused(make, "at least one element", cols=0)
    refused(make, "too long", cols=1 << 31, rows=1)
    refused(make, "too long", cols=(1 << 26) + 1, rows=1)  # a grid of the second launch counts lanes in 32 bits
    refused(make, "too many rows", rows=1 << 22)
    refused(make, "too many rows", rows=-1)
    refused(make, "too many rows", collective=RS, n=32, rows=1 << 20)
    refused(make, "stride", send_stride=63)
    refused(make, "stride", send_stride=1 << 50)
    refused(make, "eps", eps=-1e-6)
    refused(make, "eps", eps=float("nan"))
    refused(make, "send buffer is null", sendbuffs=[64 * MIB, None])
    refused(make, "element size", sendbuffs=[64 * MIB + 1, 128 * MIB])
    refused(make, "weight is null", weight=None)
    refused(make, "element size", weight=100 * 64 * MIB + 2, weight_dtype=F32)
    with pytest.raises(mr.MegRayError, match="nranks"):
        make(n=33)
    with pytest.raises(mr.MegRayError, match="nranks"):
        make(sendbuffs=[], outs=[], residuals=None, residual_outs=None) if make is forward else \
            make(sendbuffs=[], residual_out_grads=[], weight_grads=[])


def test_what_the_forward_refuses():
    refused(forward, "output's dtype", dtype=F16, out_dtype=BF16)
    refused(forward, "needs scales", out_dtype=E4M3)
    refused(forward, "scale buffer is null", out_dtype=I8, scales=[64 * MIB * 180, None])
    refused(forward, "output is null", outs=[None, 64 * MIB * 40])
    refused(forward, "2 expected", outs=buffers(3, 40))
    refused(forward, "1 expected", residuals=buffers(2, 80))
    refused(forward, "2 expected", collective=RS, residuals=buffers(1, 80))
    refused(forward, "two outputs overlap", outs=[40 * 64 * MIB] * 2)
    refused(forward, "two outputs overlap", residual_outs=buffers(2, 40))
    refused(forward, "out of place", outs=[100 * 64 * MIB, 64 * MIB * 40])  # the weight's place
    refused(forward, "two outputs overlap", out_dtype=E4M3, scales=buffers(2, 40))


def test_what_the_backward_refuses():
    refused(backward, "no gradient", residual_out_grads=None, weight_grads=None)
    refused(backward, "workspace", workspace=None)
    need = mr.rms_norm_backward_workspace(AR, 2, 4, 64)
    refused(backward, "too small", workspace_bytes=need - 1)
    backward(workspace_bytes=need)
    refused(backward, "weight gradient is null", weight_grads=[None, 64 * MIB])
    refused(backward, "overlap", workspace=120 * 64 * MIB)
    refused(backward, "overlap", weight_grads=buffers(2))
    with pytest.raises(mr.MegRayError):
        mr.rms_norm_backward_workspace(mr.Collective.BROADCAST, 2, 4, 64)
    with pytest.raises(mr.MegRayError):
        mr.rms_norm_backward_workspace(AR, 0, 4, 64)
    assert mr.rms_norm_backward_workspace(AR, 2, 0, 64) == 0


def adamw(n=2, lengths=(100, 7), **changed):
    lists = lambda first: [[b + (t << 20) for t in range(len(lengths))] for b in buffers(n, first)]  # noqa: E731
    flat = lambda first: [first * 64 * MIB + (t << 20) for t in range(len(lengths))]  # noqa: E731
    args = dict(grads=lists(1), params=lists(40), masters=flat(80), exp_avgs=flat(81), exp_avg_sqs=flat(82), param_dtype=BF16)
    args.update(changed)
    dtype = args.pop("grad_dtype", BF16)
    return mr.AdamWPlan(args.pop("grads"), list(lengths), dtype, **args)


def test_what_adamw_refuses():
    refused(adamw, "gradient dtype", grad_dtype=mr.DType.INT32)
    refused(adamw, "parameter dtype", param_dtype=E4M3)
    refused(adamw, "states are", state_dtype=F16)
    refused(adamw, "scales", state_dtype=E4M3)
    refused(adamw, "masters is null", masters=None)
    refused(adamw, "exp_avg", exp_avgs=None)
    refused(adamw, "gradient is null", grads=[[64 * MIB, None], [128 * MIB, 129 * MIB]])
    refused(adamw, "every rank has", grads=[[64 * MIB], [128 * MIB]])
    refused(adamw, "grad_ranks", grads=[])
    refused(adamw, "param_ranks", params=[])
    refused(adamw, "grad_ranks", grads=[[(1 + r) * 64 * MIB] for r in range(33)], lengths=(5,), params=None)
    refused(adamw, "overlaps", params=[[64 * MIB, 65 * MIB], [66 * 64 * MIB, 67 * 64 * MIB]])
    refused(adamw, "overlaps", exp_avgs=[82 * 64 * MIB, 81 * 64 * MIB])
    refused(adamw, "element size", exp_avgs=[81 * 64 * MIB + 2, 81 * 64 * MIB + MIB])
    refused(adamw, "weight decays", weight_decays=[0.1])
    refused(adamw, "not finite", weight_decays=[0.1, float("inf")])
    refused(adamw, "too many elements", lengths=(1 << 36,), grads=[[64 * MIB], [128 * MIB]], params=None)
    refused(adamw, "too long", lengths=(1 << 41,), grads=[[64 * MIB], [128 * MIB]], params=None)


def test_the_python_records_are_laid_out_as_the_header_says(tmp_path):
    from megray_amd import _lib

    records = {"mrv_rms_norm_call": _lib.RmsNormCall, "mrv_rms_norm_backward_call": _lib.RmsNormBackwardCall,
               "mrv_adamw_tensors": _lib.AdamwTensors, "mrv_adamw_step_args": _lib.AdamwStepArgs}
    prints = "".join(f'    printf("{c} {f} %zu\\n", offsetof({c}, {f}));\n' for c, r in records.items() for f, _ in r._fields_)
    prints += "".join(f'    printf("{c} sizeof %zu\\n", sizeof({c}));\n' for c in records)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "megray_vrank.h"\nint main(void) {{\n{prints}    return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", f"-I{os.path.join(ROOT, 'include')}",
                    str(src), "-o", str(exe)], check=True, capture_output=True, text=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        record, field, value = line.split()
        kind = records[record]
        assert int(value) == (ctypes.sizeof(kind) if field == "sizeof" else getattr(kind, field).offset), line


def test_the_new_types_are_unknown_to_every_other_call():
    for dtype in (BF16, E4M3):
        with pytest.raises(mr.MegRayError, match="unknown dtype"):
            mr.get_dtype_size(dtype)
        with pytest.raises(mr.MegRayError, match="unknown dtype"):
            mr.describe(AR, buffers(2), buffers(2, 10), 64, dtype)
