"""THHipLinear4Bit: networks whose Linear modules run with 4-bit weights on the float engines, against the same networks
with the weights that the codes stand for on the same engines, module by module."""
import subprocess

import numpy as np
import pytest

import gpu_util as G
import w4_util as U
from thnets_amd import api, configs, t7

pytestmark = pytest.mark.gpu

HALF = {G.F32: 0, G.F16: 1, G.BF16: 2}


def rounded_weights(lib, w, group, dtype):
    """What a Linear's weights are after THHipLinear4Bit(group)."""
    nOut, nIn = w.shape
    n = U.groups_of(nIn, group)
    dw = api.DeviceArray(lib, np.ascontiguousarray(w, np.float32))
    dc, ds, dz = (api.DeviceArray(lib, nbytes=k) for k in (nOut * ((nIn + 1) // 2), nOut * n * 4, nOut * n))
    assert lib.thhip_quantize_w4(dw.ptr, nIn, G.F32, dc.ptr, ds.ptr, dz.ptr, nOut, nIn, group, dtype) == 0
    lib.thhip_sync()
    layer = U.Layer(U.unpack_codes(dc.get((nOut, (nIn + 1) // 2), np.uint8), nIn),
                    U.unraw(ds.get((nOut, n), np.uint32 if dtype == G.F32 else np.uint16), dtype), dz.get((nOut, n), np.uint8), group, dtype)
    return layer.weights()


def network(g, batch):
    """Convolution, pooling and three Linear layers of sizes that nothing divides, the first two with ReLU."""
    conv = configs.conv(g.standard_normal((16, 3, 3, 3), dtype=np.float32) * np.float32(0.3), g.standard_normal(16, dtype=np.float32) * np.float32(0.1), 1, 1)

    def linear(i, o):
        return {"type": "linear", "weight": g.standard_normal((o, i), dtype=np.float32) * np.float32(np.sqrt(2.0 / i)),
                "bias": g.standard_normal(o, dtype=np.float32) * np.float32(0.1)}
    layers = [conv, configs.relu(), configs.maxpool(2, 2), {"type": "view", "numElements": 16 * 49}, linear(784, 300), configs.relu(),
              linear(300, 77), configs.relu(), linear(77, 10), {"type": "softmax"}]
    return layers, g.uniform(0, 1, (batch, 3, 14, 14)).astype(np.float32)


@pytest.mark.parametrize("dtype", [G.F32, G.F16, G.BF16])
@pytest.mark.parametrize("batch", [1, 5, 40])
@pytest.mark.parametrize("group", [32, 128])
def test_network(hiplib, group, batch, dtype):
    """The two engines see the same values in front of every Linear up to roundings of the layers before.  fp32: both sum
    fp32 products, a few 1e-6 of the largest value each.  Half types: the reference engine rounds the weights once more to
    its type (half a step each, together about half a step of the result) and both round three results; ten half
    steps bound all of it."""
    g = U.rng(3000 + group + batch)
    layers, x = network(g, batch)
    net = api.HipNetwork(layers, half=HALF[dtype], linear4=group)
    got = net.process_float(x)
    mods = [net.module_output(i) for i in (4, 6, 8)]
    assert np.array_equal(net.process_float(x), got), "the same call again"
    net.free()
    plain = [dict(s, weight=rounded_weights(hiplib, s["weight"], group, dtype).astype(np.float32)) if s["type"] == "linear" else s for s in layers]
    ref = api.HipNetwork(plain, half=HALF[dtype])
    want = ref.process_float(x)
    tol = 2e-5 if dtype == G.F32 else 10 * U.HALF_STEP[dtype]
    for i, m in zip((4, 6, 8), mods):
        G.assert_close(m, ref.module_output(i), tol, "module %d" % i)
    G.assert_close(got, want, tol, "softmax")
    ref.free()
    assert hiplib.THHipLinear4Bit(0) == 0       # (HipNetwork put the setting back)


def test_setting(hiplib):
    assert hiplib.THHipLinear4Bit(64) == 0 and hiplib.THHipLinear4Bit(7) == 64 and hiplib.THHipLinear4Bit(0) == 64
    assert hiplib.THHipLinear4Bit(0) == 0


def test_spatial_linears_are_convolutions(hiplib):
    """THMakeSpatial turns Linears into convolutions, which keep their weights: the setting changes nothing."""
    g = U.rng(3100)
    layers, x = network(g, 2)
    a, b = (api.HipNetwork(layers[:-1], make_spatial=14, linear4=q) for q in (0, 64))
    assert np.array_equal(a.process_float(x), b.process_float(x))
    a.free()
    b.free()


def test_vgg_linears(hiplib):
    """VGG-16's layer widths at an eighth, one image and four: the whole network with 4-bit Linears."""
    cfg = configs.vgg16(batch=4, scale=0.125, side=64)
    net = api.HipNetwork(cfg["layers"], linear4=128)
    got = net.process_float(cfg["input"])
    one = net.process_float(cfg["input"][:1])
    net.free()
    plain = [dict(s, weight=rounded_weights(hiplib, s["weight"], 128, G.F32).astype(np.float32)) if s["type"] == "linear" else s for s in cfg["layers"]]
    ref = api.HipNetwork(plain)
    G.assert_close(got, ref.process_float(cfg["input"]), 2e-5, "batch of four")
    G.assert_close(one, ref.process_float(cfg["input"][:1]), 2e-5, "one image")
    ref.free()


def test_other_groups_are_refused(hiplib):
    layers, _ = network(U.rng(3300), 1)
    for group in (48, -1, 512):
        with pytest.raises(ValueError):
            api.HipNetwork(layers, linear4=group)
    assert hiplib.THHipLinear4Bit(0) == 0


def test_command_line_driver(hiplib, tmp_path):
    """-q group: the driver's printed outputs are those of the engine with that setting."""
    g = U.rng(3200)
    layers, x = network(g, 1)
    d = str(tmp_path / "model")
    t7.save_model_dir(d, layers[:-1])
    t7.save(str(tmp_path / "in.t7"), x[0])
    exe = api.LIB_PATH.replace("libthnets_hip.so", "thnets-hip-test")
    out = subprocess.run([exe, "-m", d, "-i", str(tmp_path / "in.t7"), "-p", "-q", "64"], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stderr
    printed = [float(line.split(":")[1]) for line in out.stdout.splitlines() if line.startswith("(")]
    net = api.HipNetwork(d, linear4=64)
    want = net.process_float(x)
    net.free()
    assert len(printed) == want.size and np.abs(np.array(printed) - want).max() <= 1e-6 + 1e-6 * np.abs(want).max()


def test_the_setting_holds_for_networks_that_name_none(hiplib):
    """A network made without linear4 has what THHipLinear4Bit says; one made with it has its own, and the setting stays."""
    layers, x = network(U.rng(3400), 3)
    nets = [api.HipNetwork(layers, linear4=0), api.HipNetwork(layers, linear4=64)]
    assert hiplib.THHipLinear4Bit(64) == 0
    try:
        nets += [api.HipNetwork(layers), api.HipNetwork(layers, linear4=0)]
        with pytest.raises(ValueError):
            api.HipNetwork(layers, linear4=48)
        assert hiplib.THHipLinear4Bit(-1) == 64
    finally:
        hiplib.THHipLinear4Bit(0)
    plain, four, by_setting, named = (n.process_float(x) for n in nets)
    assert not np.array_equal(plain, four) and np.array_equal(by_setting, four) and np.array_equal(named, plain)
    for n in nets:
        n.free()
