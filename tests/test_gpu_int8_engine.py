"""FcnEngine(int8=...): chosen convolutions of the FCN on 8-bit integers (engine option 16 of the 16-bit engines, rcv_op::wq_off)."""
import ctypes
import json
import os

import pytest
import torch

import fcn_weights
from rcvpose_amd import _hip, fcn_engine, int8
from rcvpose_amd.fcn_engine import FcnEngine

pytestmark = pytest.mark.gpu

TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def sds(golden_dir):
    shapes = json.load(open(os.path.join(golden_dir, "fcn_state_dict_keys.json")))
    return [{k: torch.from_numpy(v) for k, v in fcn_weights.make_state_dict_numpy(shapes, seed=s).items()} for s in range(2)]


@pytest.fixture(scope="module")
def x():
    return torch.randn(3, 3, 64, 96, generator=torch.Generator().manual_seed(1)).cuda()


# one name per kind of op: long 3x3, 3x3 over two sources, a 3x3 in the middle of a bottleneck, 1x1 with and without a residual, the
# 3x3 between the last upsampling and the head
NAMES = ["conv6", "conv_up4.0", "conv_up1.0", "block2.3.conv2", "block3.7.conv1", "block4.1.conv3", "block4up.conv3", "conv7.0"]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_every_int8_op_equals_the_public_operators(sds, x, dtype):
    """The engine's op, from the stored activations: quantize_tokens + matmul / conv3x3 with the folded weights.  Groups may divide a sum
    differently (float32 additions in another order), so a value may round to the neighbouring 16-bit number."""
    eng = FcnEngine(sds, 64, 96, dtype=dtype, reuse_slots=False, int8="|".join(n.replace(".", r"\.") for n in NAMES))
    eng.forward(x)
    builder = fcn_engine.build_program(64, 96)
    seen = []
    for op, spec in zip(eng.ops, builder.wspecs):
        if not op["wq_off"]:
            continue
        seen.append(spec["conv"])
        for g in range(2):
            def get(slot, h, w, c):
                return None if slot < 0 else eng.debug_slot(3, g, slot, (h, w, c)).to(TORCH[dtype])
            src0, src1 = get(op["src0"], op["hin"], op["win"], op["c0"]), get(op["src1"], op["hin"], op["win"], op["c1"])
            res, got = get(op["res"], op["hout"], op["wout"], op["cout"]), get(op["dst"], op["hout"], op["wout"], op["cout"])
            w, b = fcn_engine.fold_conv_bn(sds[g], spec, op["cout"])
            weight = int8.quantize_weight(w[:, 0, 0] if op["ksize"] == 1 else w).to("cuda")
            call = int8.matmul if op["ksize"] == 1 else int8.conv3x3
            codes, scales = int8.quantize_tokens(src0, src1)
            want = call(codes, scales, weight, bias=b.float().cuda(), residual=res, relu=bool(op["relu"]), dtype=TORCH[dtype]).double()
            # Both are within 31 roundings of float32 (nine taps, up to sixteen partial sums, scale, bias, residual) of the same real number, a
            # rounding being at most 2^-24 of the sum of the magnitudes that are added; so they differ by twice that, and each is then
            # rounded by at most half a step of its type: eps / 2 of its value, or half of the smallest subnormal.
            size = call(codes.abs(), scales, int8.pack_codes(weight.codes[:, :, :weight.channels].abs().reshape(w.shape if op["ksize"] == 3 else w[:, 0, 0].shape),
                                                            weight.scales), bias=b.float().abs().cuda(),
                        residual=None if res is None else res.float().abs(), dtype=torch.float32).double()
            eps = torch.finfo(TORCH[dtype]).eps
            diff = (got.double() - want).abs()
            assert bool((diff <= 62 * 2.0 ** -24 * size * (1 + eps) + eps * want.abs() * (1 + eps) + 2.0 ** -24).all()), (spec["conv"], g, float(diff.max()))
            assert float((diff > 0).double().mean()) < 1e-2
            assert float(want.abs().max()) > 0
    assert sorted(seen) == sorted(NAMES)


def test_option_16_switches_back(sds, x):
    plain = FcnEngine(sds, 64, 96, dtype="bf16").forward(x)
    eng = FcnEngine(sds, 64, 96, dtype="bf16", int8=True)
    seg, rad = eng.forward(x)
    assert bool(torch.isfinite(rad).all()) and not torch.equal(rad, plain[1])
    assert float((rad - plain[1]).abs().max()) < 0.5 * float(plain[1].abs().max())
    again = eng.forward(x)
    assert torch.equal(again[0], seg) and torch.equal(again[1], rad)
    eng.set_option(16, 0)
    off = eng.forward(x)
    assert torch.equal(off[0], plain[0]) and torch.equal(off[1], plain[1])


def test_captured_forward_equals_eager(sds, x):
    eng = FcnEngine(sds, 64, 96, dtype="fp16", int8=True)
    seg, rad = [t.clone() for t in eng.forward(x)]
    graph, gs, gr = eng.capture(x)
    for _ in range(3):
        gs.zero_(), gr.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gs, seg) and torch.equal(gr, rad)
        assert torch.equal(eng.forward(x)[1], rad)
    assert eng.range_status() == 0


def test_fp16_overflow_of_an_int8_op_is_reported(sds, x):
    sd = dict(sds[0])
    sd["conv6.bias"] = sd["conv6.bias"] + 1e9  # (bn6 scales it back down, but not below 65504)
    eng = FcnEngine([sd], 64, 96, dtype="fp16", int8=r"conv6")
    eng.forward(x)
    assert eng.range_status(clear=True) & 2
    with pytest.raises(_hip.HalfRangeError):
        eng.forward(x)
        eng.range_status(raise_on_flag=True)


def test_model_and_refusals(sds, x):
    from rcvpose_amd.models.fcnresnet import DenseFCNResNet152

    m = DenseFCNResNet152(3, 2).eval()
    m.load_state_dict(sds[0])
    m.set_compute_dtype("bf16", int8=True)
    seg, rad = m(x)
    ref = FcnEngine(sds[:1], 64, 96, dtype="bf16", int8=True).forward(x)
    assert torch.equal(seg, ref[0][0]) and torch.equal(rad, ref[1][0])
    with pytest.raises(ValueError):
        FcnEngine(sds[:1], 64, 96, dtype="f16x3", int8=True)

    lib = _hip.lib()
    w = torch.zeros(1 << 16, dtype=torch.bfloat16, device="cuda")
    bias = torch.zeros(1024, device="cuda")
    base = dict(kind=_hip.OP_CONV, src0=0, src1=-1, res=-1, dst=1, c0=64, cout=64, hin=8, win=8, hout=8, wout=8, ksize=3, stride=1, pad=1, w_off=0,
                b_off=0, wq_off=40960)
    for change, status in ((dict(), _hip.RCV_OK), (dict(stride=2, hout=4, wout=4), _hip.RCV_E_UNSUPPORTED), (dict(ksize=5, pad=2), _hip.RCV_E_UNSUPPORTED),
                           (dict(pad=0, hout=6, wout=6), _hip.RCV_E_UNSUPPORTED), (dict(wq_off=40961), _hip.RCV_E_INVALID),
                           (dict(src0=_hip.SLOT_INPUT), _hip.RCV_E_INVALID)):
        op = _hip.Op(**{**base, **change})
        handle = ctypes.c_void_p()
        slots = (ctypes.c_int64 * 2)(64 * 64, 64 * 64)
        rc = lib.rcv_fcn_create(ctypes.byref(op), 1, 2, slots, 1, _hip.RCV_BF16, w.data_ptr(), bias.data_ptr(), ctypes.byref(handle))
        assert rc == status, change
        if rc == _hip.RCV_OK:
            plain = _hip.Op(**{**base, "wq_off": 0})
            h2 = ctypes.c_void_p()
            _hip.check(lib.rcv_fcn_create(ctypes.byref(plain), 1, 2, slots, 1, _hip.RCV_BF16, w.data_ptr(), bias.data_ptr(), ctypes.byref(h2)))
            # the scratch of the codes is part of the workspace: 4 images of 64 pixels x 64 codes and a scale each
            assert lib.rcv_fcn_workspace_bytes(handle, 4) >= lib.rcv_fcn_workspace_bytes(h2, 4) + 4 * 64 * (64 + 4)
            lib.rcv_fcn_destroy(h2)
            lib.rcv_fcn_destroy(handle)


def test_pipeline_runs_the_int8_engine(sds):
    """FramePipeline(int8=True): its maps are the int8 engine's, on the current stream and on a side stream."""
    from rcvpose_amd.pipeline import FramePipeline

    pipe = FramePipeline(sds, 64, 96, dtype="bf16", frames_per_step=2, int8=True)
    assert any(op["wq_off"] for op in pipe.engine.ops)
    rgb = torch.randint(0, 256, (2, 64, 96, 3), dtype=torch.uint8, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    pipe.forward_fcn(rgb)
    torch.cuda.synchronize()
    want = FcnEngine(sds, 64, 96, dtype="bf16", int8=True).forward(pipe.x)
    assert torch.equal(pipe.seg, want[0]) and torch.equal(pipe.radial, want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = pipe.engine.forward(pipe.x)
    torch.cuda.synchronize()
    assert torch.equal(again[1], want[1])


@pytest.mark.parametrize("dtype, int8", [("bf16", True), ("fp16", True), ("bf16", r"conv6|block4.*|conv_up1\.0")])
def test_a_workspace_of_a_larger_batch_serves_a_smaller_one(sds, x, dtype, int8):
    """Sums are divided where the tiles are few, so a smaller batch may need parts that a larger one does not: the workspace holds them."""
    eng = FcnEngine(sds[:1], 64, 96, dtype=dtype, int8=int8)
    sizes = [eng.workspace_bytes(b) for b in range(1, 129)]
    assert sizes == sorted(sizes)
    many = x[:1].repeat(17, 1, 1, 1)
    many.mul_(torch.linspace(0.5, 1.5, 17, device="cuda").view(17, 1, 1, 1))
    eng.forward(many)
    got = eng.forward(many[:16])
    want = FcnEngine(sds[:1], 64, 96, dtype=dtype, int8=int8).forward(many[:16])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("int8_layers", [True, r"conv6|conv_up[54321]\.0|conv7\.0|block[234](up)?(\.\d)?\.conv[123]"])
def test_an_image_alone_and_among_others(sds, x, dtype, int8_layers):
    """An image's maps are the same bits in any batch and beside any number of networks, as with 16-bit layers."""
    eng = FcnEngine(sds, 64, 96, dtype=dtype, int8=int8_layers)
    alone = [t.clone() for t in eng.forward(x[:1])]
    many = x[:1].repeat(57, 1, 1, 1)
    many[1:] *= torch.linspace(0.5, 1.5, 56, device="cuda").view(56, 1, 1, 1)
    for b in (2, 3, 8, 17, 57):
        got = eng.forward(many[:b])
        assert torch.equal(got[0][:, :1], alone[0]) and torch.equal(got[1][:, :1], alone[1]), b
    single = FcnEngine(sds[1:], 64, 96, dtype=dtype, int8=int8_layers).forward(many[:1])
    assert torch.equal(single[0][0], alone[0][1]) and torch.equal(single[1][0], alone[1][1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_a_frame_alone_and_among_others(sds, dtype):
    """The same at 480 x 640, where one frame's windows used to be added in another order than eight frames'."""
    frames = torch.randn(8, 3, 480, 640, generator=torch.Generator().manual_seed(1)).cuda()
    eng = FcnEngine(sds, 480, 640, dtype=dtype, int8=True)
    alone = [t.clone() for t in eng.forward(frames[:1])]
    for b in (2, 8):
        got = eng.forward(frames[:b])
        assert torch.equal(got[0][:, :1], alone[0]) and torch.equal(got[1][:, :1], alone[1]), b


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_keypoints_under_the_int8_engines_error(golden_dir, oracle, monkeypatch, dtype):
    """What the int8 layers' error does to the keypoints, measured as for the other types (test_gpu_pipeline: the error field of a random network,
    transferred onto ideal maps, against the fp32 engine's keypoints): the figures are printed.  What is asserted is exact: the
    device votes on the perturbed maps like the oracle, and the int8 layers' error is no smaller than the one of 16 bits they add to."""
    import numpy as np

    import test_gpu_pipeline as yard
    from rcvpose_amd import pipeline

    plain = yard._keypoints_under_engine_error(golden_dir, dtype)
    whole = pipeline.FramePipeline
    monkeypatch.setattr(pipeline, "FramePipeline", lambda *a, **kw: whole(*a, int8=kw["dtype"] != "fp32", **kw))
    dev, rel, step, (ps, pr), fr, rmax, kp = yard._keypoints_under_engine_error(golden_dir, dtype)
    for name, (d, r, s) in ((dtype, plain[:3]), (dtype + " with int8 layers", (dev, rel, step))):
        print("%s: keypoints move by %.2f voxels at most, %.3f on average, %d of %d by more than one; radial maps %s of their range (radius: max %.2f, "
              "rms %.2f voxels)" % (name, d.max(), d.mean(), int((d > 1).sum()), d.size, ["%.1e" % e for e, _ in r], s[0], s[1]))
    assert step[1] > plain[2][1]
    for b, k in ((0, 0), (3, 1), (7, 2)):
        xyz, rl = oracle.seam(ps[k, b, 0], pr[k, b, 0], fr[b]["depth"], rmax[k])
        assert np.array_equal(kp[b, k], oracle.accumulator_3d(xyz, rl, sparse=True)[0])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_res_network(golden_dir, x, dtype):
    """ResFCNResNet152: two of its decoder's windows by default, and a lateral 1x1 convolution with the upsampled tensor as its residual.  Every op
    against the public operators (the bound of test_every_int8_op_equals_the_public_operators), the model class against the engine."""
    from rcvpose_amd.models.fcnresnet import ResFCNResNet152

    shapes = json.load(open(os.path.join(golden_dir, "resfcn_state_dict_keys.json")))
    sd = {k: torch.from_numpy(v) for k, v in fcn_weights.make_state_dict_numpy(shapes, seed=0).items()}
    builder = fcn_engine.build_program_res(64, 96)
    names = ["conv_up4.0", "conv_up3.0"]
    for pattern, want_names in ((True, names), (r"conv_up[43]\.0|conv_up2_1", names + ["conv_up2_1"])):
        eng = FcnEngine([sd], 64, 96, dtype=dtype, reuse_slots=False, arch="res", int8=pattern)
        seg, rad = eng.forward(x)
        assert sorted(s["conv"] for o, s in zip(eng.ops, builder.wspecs) if o["wq_off"]) == sorted(want_names)
        for op, spec in zip(eng.ops, builder.wspecs):
            if not op["wq_off"]:
                continue
            src, got = (eng.debug_slot(3, 0, op[k], (op["hin"], op["win"], op[c])).to(TORCH[dtype]) for k, c in (("src0", "c0"), ("dst", "cout")))
            res = None if op["res"] < 0 else eng.debug_slot(3, 0, op["res"], (op["hin"], op["win"], op["cout"])).to(TORCH[dtype])
            w, b = fcn_engine.fold_conv_bn(sd, spec, op["cout"])
            weight = int8.quantize_weight(w[:, 0, 0] if op["ksize"] == 1 else w).to("cuda")
            call = int8.matmul if op["ksize"] == 1 else int8.conv3x3
            codes, scales = int8.quantize_tokens(src)
            want = call(codes, scales, weight, bias=b.float().cuda(), residual=res, relu=bool(op["relu"]), dtype=TORCH[dtype]).double()
            positive = int8.Int8Weight(weight.codes.abs(), weight.scales, weight.channels)
            size = call(codes.abs(), scales, positive, bias=b.float().abs().cuda(), residual=None if res is None else res.float().abs(), dtype=torch.float32).double()
            eps, diff = torch.finfo(TORCH[dtype]).eps, (got.double() - want).abs()
            assert bool((diff <= 62 * 2.0 ** -24 * size * (1 + eps) + eps * want.abs() * (1 + eps) + 2.0 ** -24).all()), (spec["conv"], float(diff.max()))
            assert float(want.abs().max()) > 0
    m = ResFCNResNet152(3, 2).eval()
    m.load_state_dict(sd)
    m.set_compute_dtype(dtype, int8=pattern)
    got = m(x)
    eng = FcnEngine([sd], 64, 96, dtype=dtype, arch="res", int8=pattern)
    ref = eng.forward(x)
    assert torch.equal(got[0], ref[0][0]) and torch.equal(got[1], ref[1][0])
    eng.set_option(16, 0)
    plain = FcnEngine([sd], 64, 96, dtype=dtype, arch="res").forward(x)
    off = eng.forward(x)
    assert torch.equal(off[0], plain[0]) and torch.equal(off[1], plain[1]) and not torch.equal(ref[1], plain[1])


@pytest.mark.parametrize("dtype, int8_layers", [("bf16", False), ("fp16", True)])
def test_a_graph_keeps_its_workspace(sds, x, dtype, int8_layers):
    """A forward of a larger batch gives the engine another workspace; what takes the first one's memory must not be written by a replay."""
    eng = FcnEngine(sds, 64, 96, dtype=dtype, int8=int8_layers)
    graph, seg, rad = eng.capture(x[:1])
    assert graph.workspace is eng.workspace(1)
    want = [t.clone() for t in eng.forward(x[:1])]
    size = eng.workspace(1).numel()
    eng.forward(x)
    assert graph.workspace is not eng.workspace(1)
    others = [torch.full((size,), 77, dtype=torch.uint8, device="cuda") for _ in range(3)]
    for _ in range(3):
        seg.zero_(), rad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(seg, want[0]) and torch.equal(rad, want[1])
        assert all(int((t != 77).sum()) == 0 for t in others)
