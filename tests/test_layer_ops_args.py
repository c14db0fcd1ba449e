"""What the operators around a layer's recurrence and experts refuse, before
anything is queued (no device is touched), and the workspace sizes."""
import ctypes as C

import pytest

import warp_amd.hip as wh

A = 1 << 20                                       # an aligned address that nothing reads: these calls end before a launch


def refused(fn, args, **change):
    for k, v in change.items():
        setattr(args, k, v)
    return fn(C.byref(args), None)


def no_device():
    from warp_amd.device import device_count
    return device_count() == 0


def conv():
    return wh.ConvArgs(0, 10, 3, 8, 4, A, None, 3, A, 0, A, None, 1, None, None, A + 4096, 0)


def scan():
    return wh.ScanArgs(0, 10, 3, 8, 4, 2, A, None, 3, A, 0, A, 0, A, A, A, 0, None, None, 0, None, 1, None, None, A, 0, 0,
                       None, 0)


def dispatch():
    return wh.DispatchArgs(10, 2, 8, A, A, A, A, 0, 16, A, 0, A, 0, A, 1 << 20)


def combine():
    return wh.CombineArgs(0, 10, 2, 16, A, 0, A, None, None, 0, A + 4096, 0)


def back():
    return wh.CombineBackArgs(0, 10, 2, 16, A, 0, A + 4096, 0, A, None, A + 8192, 0, A)


ROWS = [dict(type=3), dict(type=-1), dict(tokens=-1), dict(n_seq=-1), dict(channels=0), dict(channels=(1 << 24) + 1),
        dict(tokens=(1 << 30) + 1), dict(n_seq=(1 << 30) + 1, slots=A), dict(n_slots=2), dict(n_slots=-1, slots=A), dict(starts=None), dict(starts=A + 2),
        dict(slots=A + 1), dict(ldx=7), dict(ldy=7), dict(x=None), dict(y=None), dict(x=A + 2), dict(y=A + 1),
        dict(state_in=A + 2), dict(state_out=A + 2), dict(type=1, x=A + 1)]


@pytest.mark.parametrize("change", ROWS + [dict(taps=0), dict(taps=9), dict(w=None), dict(w=A + 2), dict(bias=A + 2),
                                           dict(y=A)])
def test_conv_refuses(change):
    assert refused(wh.lib().warp_hip_short_conv, conv(), **change) == wh.E_ARG


@pytest.mark.parametrize("change", ROWS + [dict(states=0), dict(states=257), dict(groups=0), dict(groups=3), dict(longest=-1),
                                           dict(lddt=7), dict(ldz=7), dict(ldbc=7), dict(A=None), dict(B=None), dict(C=None),
                                           dict(dt=None), dict(A=A + 2), dict(D=A + 2), dict(dt_bias=A + 2), dict(z=A + 2),
                                           dict(B=A + 2), dict(C=A + 2), dict(dt=A + 2)])
def test_scan_refuses(change):
    assert refused(wh.lib().warp_hip_selective_scan, scan(), **change) == wh.E_ARG


def test_scan_refuses_a_short_workspace():
    fn, need = wh.lib().warp_hip_selective_scan, wh.selective_scan_work(4096, 64, 16, 3)
    assert need > 0
    for change in (dict(), dict(work=A, work_bytes=need - 1), dict(work=A + 8, work_bytes=need)):
        assert refused(fn, scan(), tokens=4096, channels=64, states=16, **change) == wh.E_ARG


@pytest.mark.parametrize("change", [dict(tokens=-1), dict(top_k=0), dict(n_experts=0), dict(n_experts=2049), dict(idx=None),
                                    dict(offsets=None), dict(perm=None), dict(pos=None), dict(idx=A + 1), dict(offsets=A + 2),
                                    dict(perm=A + 3), dict(pos=A + 2), dict(x=None), dict(xs=None), dict(type=5),
                                    dict(hidden=0), dict(hidden=(1 << 24) + 1), dict(ldx=15), dict(ldxs=15), dict(x=A + 2),
                                    dict(xs=A + 1), dict(tokens=5000, work=None), dict(tokens=5000, work=A + 2),
                                    dict(tokens=5000, work_bytes=4), dict(tokens=(1 << 29) + 1),
                                    dict(tokens=1 << 30, top_k=2)])
def test_dispatch_refuses(change):
    assert refused(wh.lib().warp_hip_expert_dispatch, dispatch(), **change) == wh.E_ARG


@pytest.mark.parametrize("change", [dict(type=4), dict(tokens=-2), dict(top_k=0), dict(hidden=0), dict(tokens=1 << 30, top_k=2),
                                    dict(y=None), dict(pos=None), dict(out=None), dict(out=A), dict(ldy=15), dict(ldo=15),
                                    dict(resid=A, ldr=15), dict(resid=A + 4096, ldr=20), dict(y=A + 2), dict(out=A + 2),
                                    dict(resid=A + 1), dict(pos=A + 2), dict(w=A + 2)])
def test_combine_refuses(change):
    assert refused(wh.lib().warp_hip_expert_combine, combine(), **change) == wh.E_ARG


@pytest.mark.parametrize("change", [dict(type=4), dict(tokens=-2), dict(top_k=0), dict(hidden=0), dict(tokens=1 << 30, top_k=2),
                                    dict(y=None), dict(pos=None), dict(dout=None), dict(dy=None, dw=None), dict(dy=A),
                                    dict(dy=A + 4096, lddy=20), dict(ldy=15), dict(ldd=15), dict(lddy=15), dict(y=A + 2),
                                    dict(dy=A + 2), dict(dout=A + 1), dict(pos=A + 2), dict(w=A + 2), dict(dw=A + 2)])
def test_combine_backward_refuses(change):
    assert refused(wh.lib().warp_hip_expert_combine_backward, back(), **change) == wh.E_ARG


def test_null_arguments_and_calls_without_work():
    L = wh.lib()
    for fn in (L.warp_hip_short_conv, L.warp_hip_selective_scan, L.warp_hip_expert_dispatch, L.warp_hip_expert_combine,
               L.warp_hip_expert_combine_backward):
        assert fn(None, None) == wh.E_ARG
    # nothing to do: accepted without a device
    assert refused(L.warp_hip_short_conv, conv(), tokens=0, n_seq=0, x=None, y=None) == 0
    assert refused(L.warp_hip_selective_scan, scan(), tokens=0, n_seq=0, x=None, y=None) == 0
    assert refused(L.warp_hip_expert_combine, combine(), tokens=0, y=None, pos=None, out=None) == 0
    assert refused(L.warp_hip_expert_combine_backward, back(), tokens=0, dout=None, pos=None) == 0


def test_accepted_arguments_reach_the_device():
    if not no_device():
        pytest.skip("a device is present: the calls that are not refused would launch")
    L = wh.lib()
    for fn, args in ((L.warp_hip_short_conv, conv()), (L.warp_hip_selective_scan, scan()),
                     (L.warp_hip_expert_dispatch, dispatch()), (L.warp_hip_expert_combine, combine()),
                     (L.warp_hip_expert_combine_backward, back())):
        assert refused(fn, args) == wh.E_DEVICE


def test_workspace_sizes():
    assert wh.selective_scan_work(0, 64, 16, 1) == 0 and wh.selective_scan_work(64, 64, 257, 1) == 0
    assert wh.selective_scan_work(4096, 64, 16, 4096, 1) == 0          # a wave per sequence is enough
    assert wh.selective_scan_work((1 << 30) + 1, 64, 16, 1) == 0 and wh.selective_scan_work(64, (1 << 24) + 1, 16, 1) == 0
    assert wh.expert_dispatch_work(10, 2, 0) == 0 and wh.expert_dispatch_work(-1, 2, 4) == 0
    assert wh.expert_dispatch_work(10, 2, 8) >= 0


def test_python_calls_raise():
    with pytest.raises(wh.WarpHipError) as e:
        wh.short_conv(A, A, A, dtype=wh.F32, tokens=1, channels=8, taps=4, n_seq=1, n_slots=1)
    assert e.value.code == wh.E_ARG


def test_kernels_keep_to_registers(tmp_path):
    from test_kernel_scratch import READELF, scratch_bytes
    if READELF is None:
        pytest.skip("llvm-readelf not installed")
    got = {k: v for k, v in scratch_bytes(tmp_path).items() if any(n in k for n in ("k_conv_", "k_scan_", "k_sort_", "k_combine"))}
    # (k_combine_lut and k_combine_chunk are the layer's own combines)
    assert len(got) > 60 and max(v for k, v in got.items() if "lut" not in k and "chunk" not in k) == 0, got
