"""8-bit integer operators, the parts that need no GPU: weight packing and the refusals of the entry points (rcv_i8_* in
include/rcvpose_hip.h check their arguments before anything is enqueued, so the codes come back here as well)."""
import ctypes

import numpy as np
import pytest
import torch

from rcvpose_amd import _hip, int8

FAKE = 1 << 20  # an aligned address that no refused call touches


def _args(**kw):
    a = _hip.I8Args(ctypes.sizeof(_hip.I8Args), _hip.RCV_BF16, FAKE, FAKE, FAKE, FAKE, None, None, FAKE, 12, 64, 0, 32, 64, 32, 3, 4, 0, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _call(name, a):
    return getattr(_hip.load_library(), name)(ctypes.byref(a), None, 0, None)


@pytest.mark.parametrize("name", ["rcv_i8_matmul", "rcv_i8_conv3x3"])
@pytest.mark.parametrize("change, status", [
    (dict(struct_bytes=0), _hip.RCV_E_INVALID),
    (dict(out_dtype=_hip.RCV_F16X3), _hip.RCV_E_UNSUPPORTED),
    (dict(out_dtype=17), _hip.RCV_E_UNSUPPORTED),
    (dict(rows=-12), _hip.RCV_E_INVALID),
    (dict(channels=0), _hip.RCV_E_INVALID),
    (dict(out_channels=0), _hip.RCV_E_INVALID),
    (dict(channels=131072, codes_pitch=131072), _hip.RCV_E_TOO_LARGE),
    (dict(codes=None), _hip.RCV_E_INVALID),
    (dict(code_scales=None), _hip.RCV_E_INVALID),
    (dict(weights=None), _hip.RCV_E_INVALID),
    (dict(weight_scales=None), _hip.RCV_E_INVALID),
    (dict(out=None), _hip.RCV_E_INVALID),
    (dict(codes=FAKE + 4), _hip.RCV_E_INVALID),
    (dict(weights=FAKE + 8), _hip.RCV_E_INVALID),
    (dict(out=FAKE + 1), _hip.RCV_E_INVALID),
    (dict(codes_pitch=72), _hip.RCV_E_INVALID),
    (dict(codes_pitch=48), _hip.RCV_E_INVALID),
    (dict(out_pitch=31), _hip.RCV_E_INVALID),
    (dict(residual=FAKE, residual_pitch=31), _hip.RCV_E_INVALID),
    (dict(residual=FAKE + 1, residual_pitch=32), _hip.RCV_E_INVALID),
    (dict(codes_pitch=1 << 23), _hip.RCV_E_TOO_LARGE),
    (dict(out_pitch=1 << 25), _hip.RCV_E_TOO_LARGE),
])
def test_product_refuses(name, change, status):
    assert _call(name, _args(**change)) == status


def test_conv_refuses_rows_that_are_no_images():
    assert _call("rcv_i8_conv3x3", _args(rows=13)) == _hip.RCV_E_INVALID
    assert _call("rcv_i8_conv3x3", _args(height=0)) == _hip.RCV_E_INVALID
    assert _call("rcv_i8_conv3x3", _args(width=-4)) == _hip.RCV_E_INVALID
    assert _call("rcv_i8_conv3x3", _args(height=1, width=1 << 17, rows=1 << 17)) == _hip.RCV_E_TOO_LARGE


def test_no_rows_is_no_work():
    for name in ("rcv_i8_matmul", "rcv_i8_conv3x3"):
        assert _call(name, _args(rows=0)) == _hip.RCV_OK
        assert getattr(_hip.load_library(), name + "_workspace_bytes")(0, 64, 32) == 0
    assert _hip.load_library().rcv_i8_quantize_tokens(FAKE, 64, 64, None, 0, 0, _hip.RCV_F32, 0, FAKE, 64, FAKE, None) == _hip.RCV_OK


@pytest.mark.parametrize("bad, status", [
    (dict(x0=None), _hip.RCV_E_INVALID), (dict(c0=0), _hip.RCV_E_INVALID), (dict(c1=-1), _hip.RCV_E_INVALID),
    (dict(c1=8, x1=None), _hip.RCV_E_INVALID), (dict(rows=-1), _hip.RCV_E_INVALID), (dict(codes=None), _hip.RCV_E_INVALID),
    (dict(scales=None), _hip.RCV_E_INVALID), (dict(dtype=_hip.RCV_F16X3), _hip.RCV_E_UNSUPPORTED), (dict(pitch0=63), _hip.RCV_E_INVALID),
    (dict(c1=8, x1=FAKE, pitch1=7, codes_pitch=72), _hip.RCV_E_INVALID), (dict(codes_pitch=63), _hip.RCV_E_INVALID),
    (dict(c0=131072, pitch0=131072, codes_pitch=131072), _hip.RCV_E_TOO_LARGE), (dict(x0=FAKE + 1), _hip.RCV_E_INVALID),
])
def test_quantize_refuses(bad, status):
    a = dict(x0=FAKE, pitch0=64, c0=64, x1=None, pitch1=0, c1=0, dtype=_hip.RCV_BF16, rows=4, codes=FAKE, codes_pitch=64, scales=FAKE)
    a.update(bad)
    assert _hip.load_library().rcv_i8_quantize_tokens(*a.values(), None) == status


@pytest.mark.parametrize("shape", [(1, 1), (5, 128), (7, 129), (6, 3, 3, 20)])
def test_weight_quantisation(shape):
    rng = np.random.default_rng(3)
    w = rng.standard_normal(shape).astype(np.float32) * np.exp(rng.standard_normal((shape[0],) + (1,) * (len(shape) - 1))).astype(np.float32)
    w[0] = 0
    q = int8.quantize_weight(torch.from_numpy(w))
    taps = 1 if len(shape) == 2 else 9
    assert tuple(q.codes.shape) == (shape[0], taps, -(-shape[-1] // 128) * 128) and q.channels == shape[-1]
    assert int(q.codes[:, :, shape[-1]:].abs().sum()) == 0
    s = (np.abs(w.reshape(shape[0], -1)).max(axis=1).astype(np.float64) / 127).astype(np.float32)
    np.testing.assert_array_equal(q.scales.numpy(), s)
    ref = np.round(w.reshape(shape[0], -1).astype(np.float64) / np.where(s > 0, s, 1)[:, None].astype(np.float64)).reshape(shape)
    np.testing.assert_array_equal(q.codes[:, :, :shape[-1]].numpy().reshape(shape), ref.astype(np.int8))
    # a code is at most half a step away (plus float32's rounding of code * scale)
    lim = s.reshape((-1,) + (1,) * (len(shape) - 1)) * (0.5 + 127 * 2.0 ** -23)
    assert (np.abs(q.dequantize().numpy() - w) <= lim).all()


def test_weight_refusals():
    with pytest.raises(ValueError):
        int8.quantize_weight(torch.tensor([[1.0, float("nan")]]))
    with pytest.raises(ValueError):
        int8.quantize_weight(torch.ones(4, 2, 3, 3))  # channels first
    with pytest.raises(ValueError):
        int8.quantize_weight(torch.ones(4, 4, dtype=torch.int32))
    with pytest.raises(ValueError):
        int8.pack_codes(torch.ones(4, 4), torch.ones(4))
    with pytest.raises(ValueError):
        int8.pack_codes(torch.ones(4, 4, dtype=torch.int8), torch.ones(3))
    with pytest.raises(ValueError):
        int8.pack_codes(torch.ones(0, 4, dtype=torch.int8), torch.ones(0))
    with pytest.raises(ValueError):
        int8.pack_codes(torch.ones(1, 131072, dtype=torch.int8), torch.ones(1))


def test_packed_weight_refusals():
    """A weight put together by hand has to have the layout that the kernels read."""
    good = int8.pack_codes(torch.ones(8, 40, dtype=torch.int8), torch.ones(8))
    int8.Int8Weight(good.codes, good.scales, 40)
    for codes, scales, channels in ((good.codes.float(), good.scales, 40), (good.codes[:, 0], good.scales, 40), (good.codes, good.scales, 129),
                                    (good.codes, good.scales, 0), (good.codes[:, :, :64], good.scales, 40),
                                    (good.codes.expand(8, 2, 128).contiguous(), good.scales, 40), (good.codes.expand(8, 9, 128), good.scales, 40),
                                    (good.codes[:0], good.scales[:0], 40), (good.codes, good.scales[:7], 40), (good.codes, good.scales.double(), 40),
                                    (good.codes, torch.ones(16)[::2], 40)):
        with pytest.raises(ValueError):
            int8.Int8Weight(codes, scales, channels)


def test_more_rows_than_a_launch_has_threads_for_are_refused():
    assert _call("rcv_i8_matmul", _args(rows=(1 << 30) + 1)) == _hip.RCV_E_TOO_LARGE
    assert _call("rcv_i8_conv3x3", _args(rows=12 << 28)) == _hip.RCV_E_TOO_LARGE


def test_no_cpu_fallback():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    with pytest.raises(_hip.HipLibraryError):
        int8.quantize_tokens(torch.ones(2, 4))
    with pytest.raises(_hip.HipLibraryError):
        int8.matmul(torch.ones(2, 4, dtype=torch.int8), torch.ones(2), int8.quantize_weight(torch.ones(3, 4)))


def test_engine_weights_with_an_int8_copy():
    """pack_weights(int8=...): codes and scales of the matching convolutions behind the 16-bit copy, every other op as without."""
    import json
    import os

    import fcn_weights
    from rcvpose_amd import fcn_engine

    golden = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")
    shapes = json.load(open(os.path.join(golden, "fcn_state_dict_keys.json")))
    sds = [{k: torch.from_numpy(v) for k, v in fcn_weights.make_state_dict_numpy(shapes, seed=s).items()} for s in range(2)]
    b = fcn_engine.build_program(64, 96)
    names = ["conv_up3.0", "block4.1.conv3"]
    w0, b0, ops0 = fcn_engine.pack_weights(sds, b, fcn_engine.assign_slots(b)[0], _hip.RCV_BF16)
    w1, b1, ops1 = fcn_engine.pack_weights(sds, b, fcn_engine.assign_slots(b)[0], _hip.RCV_BF16, int8="|".join(n.replace(".", r"\.") for n in names))
    seen = []
    for o0, o1, spec in zip(ops0, ops1, b.wspecs):
        assert o0["wq_off"] == 0
        if spec is None:
            continue
        k = o1["c0"] + (o1["c1"] if o1["src1"] >= 0 else 0)
        n_w = 2 * o1["cout"] * o1["ksize"] ** 2 * k
        assert torch.equal(w0[o0["w_off"]:o0["w_off"] + n_w].view(torch.int16), w1[o1["w_off"]:o1["w_off"] + n_w].view(torch.int16))
        assert torch.equal(b0[o0["b_off"]:o0["b_off"] + 2 * o1["cout"]], b1[o1["b_off"]:o1["b_off"] + 2 * o1["cout"]])
        if spec["conv"] not in names:
            assert o1["wq_off"] == 0
            continue
        seen.append(spec["conv"])
        taps, kp = o1["ksize"] ** 2, -(-k // 128) * 128
        assert o1["wq_off"] % 8 == 0
        codes = w1[o1["wq_off"]:o1["wq_off"] + o1["cout"] * taps * kp].view(torch.int8).view(2, o1["cout"], taps, kp)
        scales = b1[o1["b_off"] + 2 * o1["cout"]:o1["b_off"] + 4 * o1["cout"]].view(2, o1["cout"])
        for g in range(2):
            w, _ = fcn_engine.fold_conv_bn(sds[g], spec, o1["cout"])
            q = int8.quantize_weight(w[:, 0, 0] if taps == 1 else w)
            assert torch.equal(codes[g], q.codes) and torch.equal(scales[g], q.scales)
    assert sorted(seen) == sorted(names)
    # the split-precision engine's second copies stay what they are
    assert fcn_engine.pack_weights(sds[:1], b, fcn_engine.assign_slots(b)[0], _hip.RCV_F16X3, int8=True)[0].numel() == \
        fcn_engine.pack_weights(sds[:1], b, fcn_engine.assign_slots(b)[0], _hip.RCV_F16X3)[0].numel()


def test_model_takes_int8_with_16_bit_types_only():
    from rcvpose_amd.models.fcnresnet import DenseFCNResNet152

    m = DenseFCNResNet152(3, 2)
    assert m.set_compute_dtype("bf16", int8=True).int8 is True
    assert m.set_compute_dtype("fp16").int8 is False
    for name in ("f16x3", "fp32"):
        with pytest.raises(ValueError):
            m.set_compute_dtype(name, int8=True)
    assert m.compute_dtype == "fp16"


def test_main_takes_int8():
    from rcvpose_amd import main

    assert main.build_parser().parse_args([]).int8 is False
    opts = main.build_parser().parse_args(["--dtype", "bf16", "--int8", "true"])
    assert opts.int8 is True and opts.dtype == "bf16"


def test_workspace_bounds():
    """The partial sums of a divided product: at most 2^24 bytes, and at most what an engine reserves for a layer whatever the batch (nine
    parts of a window, for a product eight or one per eight steps of 128 channels).  The sums of one batch may be divided where those
    of a larger one are not."""
    lib = _hip.load_library()
    rng = np.random.default_rng(2)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))
    sizes = [(log(1, 1 << 20), log(1, 131071), log(1, 1 << 16)) for _ in range(20000)]
    sizes += [(rows, k, n) for k, n in ((131071, 1), (131071, 100), (131071, 1000), (20000, 1300), (2048, 1024), (512, 64)) for rows in range(1, 2000)]
    divided = 0
    for taps, name in ((1, "rcv_i8_matmul_workspace_bytes"), (9, "rcv_i8_conv3x3_workspace_bytes")):
        fn = getattr(lib, name)
        for rows, k, n in sizes:
            need = fn(rows, k, n)
            divided += need > 0
            parts = 9 if taps == 9 else max(8, -(-k // 128) // 8)
            assert need <= min(1 << 24, parts * rows * -(-n // 4) * 16), (taps, rows, k, n)
    assert divided > 1000
    assert lib.rcv_i8_conv3x3_workspace_bytes(2000, 1024, 1024) < lib.rcv_i8_conv3x3_workspace_bytes(500, 1024, 1024)


@pytest.mark.parametrize("shape", [(8, 40), (5, 3, 3, 130)])
def test_packed_weight_with_codes_behind_its_channels_is_refused(shape):
    """They would meet whatever lies behind a token's last code."""
    good = int8.pack_codes(torch.ones(shape, dtype=torch.int8), torch.ones(shape[0]))
    k = shape[-1]
    int8.Int8Weight(good.codes.clone(), good.scales, k)
    for at in ((0, 0, k), (shape[0] - 1, good.taps - 1, good.codes.shape[2] - 1)):
        codes = good.codes.clone()
        codes[at] = -1
        with pytest.raises(ValueError):
            int8.Int8Weight(codes, good.scales, k)
    int8.Int8Weight(torch.ones(4, 1, 128, dtype=torch.int8), torch.ones(4), 128)  # (no padding to look at)


def test_weights_of_a_parameter_hold_no_graph():
    w = torch.nn.Parameter(torch.randn(6, 20))
    q = int8.quantize_weight(w)
    assert not q.scales.requires_grad and q.scales.grad_fn is None and not q.dequantize().requires_grad
    assert torch.equal(q.scales, int8.quantize_weight(w.detach()).scales)
    p = int8.pack_codes(torch.ones(6, 20, dtype=torch.int8), torch.ones(6, requires_grad=True) * 2)
    assert not p.scales.requires_grad


@pytest.mark.parametrize("shape", [(0, 16), (4, 0), (0, 3, 3, 16), (4, 3, 3, 0)])
def test_weights_without_a_row_or_a_channel_are_refused(shape):
    with pytest.raises(ValueError):
        int8.quantize_weight(torch.ones(shape))


@pytest.mark.parametrize("name", ["rcv_i8_matmul", "rcv_i8_conv3x3"])
@pytest.mark.parametrize("field", ["code_scales", "weight_scales", "bias"])
def test_product_refuses_numbers_off_their_alignment(name, field):
    for off in (1, 2, 3):
        assert _call(name, _args(rows=0, **{field: FAKE + off})) == _hip.RCV_E_INVALID
    assert _call(name, _args(rows=0, **{field: FAKE + 4})) == _hip.RCV_OK


def test_quantize_refuses_scales_off_their_alignment():
    for off, status in ((2, _hip.RCV_E_INVALID), (4, _hip.RCV_OK)):
        assert _hip.load_library().rcv_i8_quantize_tokens(FAKE, 64, 64, None, 0, 0, _hip.RCV_F32, 0, FAKE, 64, FAKE + off, None) == status


@pytest.mark.parametrize("arch", ["dense", "res"])
def test_a_pattern_that_names_no_convolution_is_refused(arch):
    """A misspelt layer would leave an engine without an int8 layer; so would names whose convolutions the integer kernels do not run."""
    from rcvpose_amd import fcn_engine

    b = (fcn_engine.build_program if arch == "dense" else fcn_engine.build_program_res)(64, 96)
    ops = fcn_engine.assign_slots(b)[0]
    for pattern in ("typo", "conv_up4", r"conv1", r"block2up\.conv2"):
        for dtype in (_hip.RCV_BF16, _hip.RCV_F16):
            with pytest.raises(ValueError, match="int8"):
                fcn_engine.pack_weights([], b, ops, dtype, int8=pattern)


@pytest.mark.parametrize("dtype", [None, "f16x3", "fp32"])
def test_commands_refuse_int8_with_other_types(dtype, capsys):
    """The bench dropped the flag silently, main.py went as far as building the engine."""
    import bench
    from rcvpose_amd import main

    extra = [] if dtype is None else ["--dtype", dtype]
    with pytest.raises(SystemExit):
        bench.parse(["--int8"] + extra)
    with pytest.raises(SystemExit, match="int8"):
        main.main(["--int8", "true", "--mode", "test"] + extra)
    capsys.readouterr()
    assert bench.parse(["--int8", "--dtype", "fp16"]).int8 is True and bench.parse([]).int8 is False


def test_pipeline_refuses_int8_for_an_engine_that_is_built():
    from rcvpose_amd.pipeline import FramePipeline

    with pytest.raises(ValueError, match="int8"):
        FramePipeline([{}], 64, 96, dtype="bf16", fcn=object(), int8=True)


@pytest.mark.parametrize("name", ["rcv_i8_matmul", "rcv_i8_conv3x3"])
@pytest.mark.parametrize("rows, k, n", [(5, 2 ** 31 - 1, 64), (5, 131072, 64), (2 ** 62, 4096, 64), ((1 << 32) + 1, 4096, 64), (5, 4096, 2 ** 31 - 1),
                                        (5, 4096, (1 << 20) + 1), (-5, 4096, 64), (5, -4096, 64), (5, 4096, -64)])
def test_sizes_that_are_refused_need_no_workspace(name, rows, k, n):
    """(What the plan of such a size would need cannot be counted in its integers.)"""
    assert getattr(_hip.load_library(), name + "_workspace_bytes")(rows, k, n) == 0


def test_a_module_saved_before_it_had_int8_layers_runs_without():
    import copy

    from rcvpose_amd.models.fcnresnet import DenseFCNResNet152, ResFCNResNet152

    for cls in (DenseFCNResNet152, ResFCNResNet152):
        state = cls(3, 2).__dict__.copy()
        state.pop("int8", None)
        m = cls.__new__(cls)
        m.__setstate__(state)
        assert m.int8 is False and m.compute_dtype == "f16x3"
        assert copy.copy(m.set_compute_dtype("bf16", int8=True)).int8 is True
