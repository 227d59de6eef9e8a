"""What the entry points of 4-bit layers and of norms with 8-bit outputs refuse: before anything touches a GPU, with -1
and a message; and that no rows are no launch.  Runs without a GPU: the pointers are never followed."""
import os
import subprocess

import pytest

from thnets_amd import abi, api

F32, F16, BF16, U8 = abi.THHIP_F32, abi.THHIP_F16, abi.THHIP_BF16, abi.THHIP_U8
P = 1 << 20     # an aligned address


@pytest.fixture(scope="module")
def lib():
    return api.load_library()


def test_packed_bytes(lib):
    # 16-row blocks x steps of 128: 1 KiB each; 16 scales a block and group; 16 zeros; 16 bytes more
    assert lib.thhip_w4_packed_bytes(16, 128, 128, F16, 0) == 1024 + 32
    assert lib.thhip_w4_packed_bytes(17, 129, 128, F16, 1) == 4 * 1024 + 2 * 2 * 32 + 2 * 2 * 16
    assert lib.thhip_w4_packed_bytes(16, 4096, 0, F32, 0) == 32 * 1024 + 64
    assert lib.thhip_w4_packed_bytes(1, 1, 32, BF16, 1) == 1024 + 32 + 16
    # beyond 32 bits
    assert lib.thhip_w4_packed_bytes(1 << 20, 1 << 20, 0, F16, 0) == (1 << 39) + (1 << 21)
    for bad in ((0, 128, 128, F16, 0), (16, 0, 128, F16, 0), (16, 128, 48, F16, 0), (16, 128, 512, F16, 0), (16, 128, -32, F16, 0),
                (16, 128, 128, U8, 0), (16, 128, 128, 7, 0), ((1 << 30) + 1, 128, 128, F16, 0)):
        assert lib.thhip_w4_packed_bytes(*bad) == 0, bad


LINEAR = dict(x=P, ldx=256, w=P, bias=P, y=P, ldy=64, B=3, nIn=256, nOut=64, group=128, zeros=0, act=0, thr=0.0, val=0.0, dtype=F16)


@pytest.mark.parametrize("change,says", [
    (dict(x=None), "needed"), (dict(w=None), "needed"), (dict(y=None), "needed"),
    (dict(B=-1), "rows"), (dict(nIn=0), "inputs"), (dict(nOut=0), "outputs"), (dict(nIn=-5), "inputs"),
    (dict(ldx=255), "stride"), (dict(ldy=63), "stride"), (dict(group=16), "group"), (dict(group=96), "group"),
    (dict(dtype=U8), "type"), (dict(dtype=-1), "type"), (dict(x=P + 1), "aligned"), (dict(y=P + 1), "aligned"),
    (dict(w=P + 8), "aligned"), (dict(bias=P + 2), "aligned"), (dict(dtype=F32, x=P + 2), "aligned"),
])
def test_linear_refuses(lib, capfd, change, says):
    a = dict(LINEAR, **change)
    assert lib.thhip_linear_w4(*a.values()) == -1
    err = capfd.readouterr().err
    assert "thhip_linear_w4:" in err and says in err
    if not {"x", "dtype"} & set(change) or change == dict(x=None):      # (codes are bytes)
        del a["x"], a["ldx"]
        assert lib.thhip_linear_w4_i8(change.get("x", P), change.get("ldx", 256), P, 0, *a.values()) == -1
        assert says in capfd.readouterr().err


@pytest.mark.parametrize("xscale,xgroup,says", [(None, 0, "needed"), (P, 64, "scales of x"), (P, -1, "scales of x"), (P + 2, 0, "aligned")])
def test_linear_i8_refuses(lib, capfd, xscale, xgroup, says):
    a = dict(LINEAR)
    del a["x"], a["ldx"]
    assert lib.thhip_linear_w4_i8(P, 256, xscale, xgroup, *a.values()) == -1
    assert says in capfd.readouterr().err


def test_no_rows(lib):
    a = dict(LINEAR, B=0, x=None, y=None)
    assert lib.thhip_linear_w4(*a.values()) == 0
    assert lib.thhip_rmsnorm(None, 64, None, 64, None, 1e-5, None, 64, None, 64, 0, 64, F16) == 0
    assert lib.thhip_rmsnorm_i8(None, 64, None, 64, None, 1e-5, None, 64, None, 64, None, 32, 0, 64, F16) == 0
    assert lib.thhip_quantize_rows(None, 64, None, 64, None, 32, 0, 64, F16) == 0
    assert lib.thhip_dequantize_rows(None, 64, None, 32, None, 64, 0, 64, F16) == 0


@pytest.mark.parametrize("args,says", [
    ((None, P, None, P, 16, 64, 32, F16), "needed"), ((P, None, None, P, 16, 64, 32, F16), "needed"),
    ((P, P, None, None, 16, 64, 32, F16), "needed"), ((P, P, None, P + 4, 16, 64, 32, F16), "aligned"),
    ((P, P, None, P, 16, 64, 33, F16), "group"), ((P, P, None, P, 16, 64, 32, U8), "type"), ((P, P, None, P, 0, 64, 32, F16), "outputs"),
])
def test_pack_refuses(lib, capfd, args, says):
    assert lib.thhip_w4_pack(*args) == -1
    assert says in capfd.readouterr().err


@pytest.mark.parametrize("args,says", [
    ((None, 64, F32, P, P, None, 16, 64, 32, F16), "needed"), ((P, 63, F32, P, P, None, 16, 64, 32, F16), "stride"),
    ((P, 64, U8, P, P, None, 16, 64, 32, F16), "weights"), ((P, 64, F32, P, P, None, 16, 64, 8, F16), "group"),
    ((P, 64, F32, P, P, None, 16, 64, 32, U8), "type"),
])
def test_quantize_refuses(lib, capfd, args, says):
    assert lib.thhip_quantize_w4(*args) == -1
    assert says in capfd.readouterr().err


NORM = dict(x=P, ldx=64, res=P, ldr=64, w=P, eps=1e-5, sum=P, lds=64, y=P, ldy=64, rows=4, cols=64, dtype=F16)


@pytest.mark.parametrize("change,says", [
    (dict(x=None), "needed"), (dict(y=None), "needed"), (dict(rows=-1), "rows"), (dict(cols=0), "columns"), (dict(cols=1 << 31, ldx=1 << 32), "columns"),
    (dict(ldx=63), "stride"), (dict(ldr=63), "stride"), (dict(lds=63), "stride"), (dict(ldy=63), "stride"),
    (dict(dtype=U8), "type"), (dict(x=P + 1), "aligned"), (dict(res=P + 1), "aligned"), (dict(w=P + 2), "aligned"), (dict(sum=P + 1), "aligned"),
])
def test_norm_refuses(lib, capfd, change, says):
    a = dict(NORM, **change)
    assert lib.thhip_rmsnorm(*a.values()) == -1
    assert says in capfd.readouterr().err
    v = list(a.values())
    assert lib.thhip_rmsnorm_i8(*v[:10], P, 32, *v[10:]) == -1
    assert says in capfd.readouterr().err


def test_codes_refuse(lib, capfd):
    for group in (16, 48, 512, -32):
        assert lib.thhip_quantize_rows(P, 64, P, 64, P, group, 4, 64, F16) == -1
        assert "group" in capfd.readouterr().err
    assert lib.thhip_quantize_rows(P, 64, P, 63, P, 32, 4, 64, F16) == -1
    assert "stride" in capfd.readouterr().err
    assert lib.thhip_quantize_rows(P, 64, P, 64, None, 32, 4, 64, F16) == -1
    assert lib.thhip_dequantize_rows(P, 64, P, 32, None, 64, 4, 64, F16) == -1
    assert lib.thhip_dequantize_rows(None, 64, P, 32, P, 64, 4, 64, F16) == -1


def test_the_driver_refuses_other_groups():
    exe = os.path.join(os.path.dirname(api.LIB_PATH), "thnets-hip-test")
    out = subprocess.run([exe, "-m", "nowhere", "-i", "random", "-q", "48"], capture_output=True, text=True, timeout=60)
    assert out.returncode and out.stderr.startswith("Syntax")


def test_the_uint8_engine_has_no_4_bit_weights():
    exe = os.path.join(os.path.dirname(api.LIB_PATH), "thnets-hip-test")
    out = subprocess.run([exe, "-m", "nowhere", "-i", "random", "-a", "11", "-q", "64"], capture_output=True, text=True, timeout=60)
    assert out.returncode and out.stderr.startswith("Syntax")
    with pytest.raises(ValueError, match="uint8"):
        api.HipNetwork([], lowp_range=4.0, linear4=64)
