"""8-bit integer products with one scale per token and one per output channel (rcv_i8_* in include/rcvpose_hip.h).

    weight = quantize_weight(w)                          # once: [N, K], or a 3x3 convolution's [N, 3, 3, C] (channels last)
    codes, scales = quantize_tokens(x)                   # x [..., C], float32 / bfloat16 / float16
    y = matmul(codes, scales, weight, bias, relu=True)   # [..., N]
    y = conv3x3(codes, scales, weight, bias)             # codes [B, H, W, C] -> [B, H, W, N], zero padding, stride 1

A token is one row of a channels-last tensor; its value is codes * scale.  FcnEngine(int8=...) runs chosen convolutions of the FCN on
these kernels.  Inference only: no gradient flows through; there is no CPU fallback.  Results do not depend on the run: integer sums are exact and float sums
have an order that the sizes alone decide (matmul gives a token the same bits in any batch; conv3x3's nine taps may be added in another
order in a batch of another size, so that the last bits of the float32 sum differ and its rounding to 16 bits may fall to the other side).
The reference has no counterpart (its forward is fp32, models/fcnresnet.py:121-191).
"""
import ctypes
import struct

import torch

from . import _hip

KP = 128  # weight rows are zero-padded to a multiple of this many codes per tap (include/rcvpose_hip.h)
MAX_CHANNELS = 131071
_ARGS_BYTES = ctypes.sizeof(_hip.I8Args)
_pack_args = struct.Struct("@Ii7P4q6i").pack  # struct rcv_i8_args (a ctypes structure takes a microsecond longer to fill)
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_DTYPES = {torch.float32: _hip.RCV_F32, torch.bfloat16: _hip.RCV_BF16, torch.float16: _hip.RCV_F16}


class Int8Weight:
    """Packed weights of one layer: `codes` int8 [N, taps, K padded with zeros to a multiple of 128], `scales` float32 [N].
    taps is 1 (matmul) or 9 (conv3x3).  The padding is looked at once, here: what lies behind a token's last code is anything, and only
    zeros keep it out of the sums."""

    def __init__(self, codes, scales, channels, _padded=False):
        if (codes.dtype != torch.int8 or codes.dim() != 3 or codes.shape[0] == 0 or codes.shape[1] not in (1, 9) or not codes.is_contiguous() or
                not 1 <= channels <= MAX_CHANNELS or codes.shape[2] != (channels + KP - 1) // KP * KP):
            raise ValueError("packed weight codes must be contiguous int8 [N, 1 or 9, channels padded to a multiple of %d]: see pack_codes" % KP)
        if scales.dtype != torch.float32 or tuple(scales.shape) != (codes.shape[0],) or not scales.is_contiguous() or scales.device != codes.device:
            raise ValueError("weight scales must be contiguous float32 [N] on the codes' device")
        if not _padded and bool(codes[:, :, channels:].any()):
            raise ValueError("packed weight codes must be zero behind their %d channels: see pack_codes" % channels)
        self.codes, self.scales, self.channels = codes, scales, channels
        self.out_channels, self.taps = int(codes.shape[0]), int(codes.shape[1])

    def to(self, device):
        return Int8Weight(self.codes.to(device), self.scales.to(device), self.channels, _padded=True)

    def dequantize(self):
        """float32 [N, K] or [N, 3, 3, C]: the values the codes stand for."""
        v = self.codes[:, :, :self.channels].float() * self.scales.view(-1, 1, 1)
        return v[:, 0] if self.taps == 1 else v.view(self.out_channels, 3, 3, self.channels)


def pack_codes(codes, scales):
    """Int8Weight from codes [N, K] or [N, 3, 3, C] (int8) and one scale per output channel (float32 [N]), on the codes' device."""
    if codes.dtype != torch.int8 or codes.dim() not in (2, 4) or (codes.dim() == 4 and tuple(codes.shape[1:3]) != (3, 3)):
        raise ValueError("weight codes must be int8 [N, K] or [N, 3, 3, C]")
    if scales.dtype != torch.float32 or tuple(scales.shape) != (codes.shape[0],) or scales.device != codes.device:
        raise ValueError("weight scales must be float32 [N] on the codes' device")
    scales = scales.detach()
    n, k = codes.shape[0], codes.shape[-1]
    if n == 0 or k == 0 or k > MAX_CHANNELS:
        raise ValueError("an int8 weight needs at least one row and 1 ... %d channels" % MAX_CHANNELS)
    taps = 1 if codes.dim() == 2 else 9
    packed = torch.zeros(n, taps, (k + KP - 1) // KP * KP, dtype=torch.int8, device=codes.device)
    packed[:, :, :k] = codes.reshape(n, taps, k)
    return Int8Weight(packed, scales.contiguous(), int(k), _padded=True)


def quantize_weight(w):
    """Float weights [N, K] or [N, 3, 3, C] -> Int8Weight: one scale per output channel, max |w| / 127, codes rounded half to even
    (in float64, on w's device: done once per layer).  A channel of zeros gets scale 0; non-finite weights raise ValueError."""
    if not w.is_floating_point() or w.dim() not in (2, 4):
        raise ValueError("weights must be floating point [N, K] or [N, 3, 3, C]")
    if w.numel() == 0:
        raise ValueError("an int8 weight needs at least one row and 1 ... %d channels" % MAX_CHANNELS)
    w = w.detach()  # (a layer's parameter: the scales must not hold its graph)
    flat = w.reshape(w.shape[0], -1).double()
    if not bool(torch.isfinite(flat).all()):
        raise ValueError("weights are not finite")
    scales = (flat.abs().amax(dim=1) / 127).float()
    scales = torch.where(scales < 2.0 ** -126, torch.zeros_like(scales), scales)
    if not bool(torch.isfinite(scales).all()):
        raise ValueError("weights are beyond float32's range")
    safe = torch.where(scales > 0, scales, torch.ones_like(scales)).double()
    codes = torch.where(scales[:, None] > 0, torch.round(flat / safe[:, None]), torch.zeros_like(flat))
    return pack_codes(codes.clamp_(-127, 127).to(torch.int8).view(w.shape), scales)


def _rows(t, border=1, farthest=1 << 24):
    """A channels-last tensor as (tensor, number of rows, row pitch in elements); anything whose leading dimensions do not walk rows at
    one pitch of up to `farthest` is copied, to rows that start a multiple of `border` elements apart (rows that overlap: one behind the other)."""
    c = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // c if c else 0, c
    if c == 1 or t.stride(-1) == 1:
        rows, pitch, uniform = 1, None, True
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if pitch is None:
                pitch = stride
            elif stride != pitch * rows:
                uniform = False
            rows *= size
        pitch = c if pitch is None else pitch
        if uniform and c <= pitch <= farthest:
            return t, rows, pitch
        if uniform and 0 < pitch < c:
            border = 1
    pitch = (c + border - 1) // border * border
    copy = t.contiguous() if pitch == c else torch.empty(*t.shape[:-1], pitch, dtype=t.dtype, device=t.device)[..., :c].copy_(t)
    return copy, t.numel() // c, pitch


def _elsewhere(t):
    """The error for a tensor that is not where the call's first tensor is."""
    if not t.is_cuda:
        _hip.lib()  # (raises first where no GPU is visible)
        raise RuntimeError("rcvpose_amd runs on MI355X only: move the tensors to 'cuda' (no CPU fallback)")
    raise ValueError("all tensors of a call must be on one device")


def _call(index, name, fn, *args):
    """fn(*args, stream) on device `index`'s current stream."""
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _hip.check(rc, name)


def quantize_tokens(x, x1=None):
    """x [..., C] (float32, bfloat16 or float16), optionally a second tensor [..., C1] of the same type whose channels follow (the
    concatenation is not materialised) -> (codes int8 [..., C + C1], scales float32 [...]).

    scale = float32(max |x| / 127) of the token, code = x / scale rounded half to even.  A token of zeros gets scale 0; a token with a
    NaN or an infinity gets scale NaN and codes 0, so products with it are NaN.  The rows of `codes` start 16 bytes aligned, as
    matmul and conv3x3 need them: for C not a multiple of 16 `codes` is a view of a wider buffer."""
    L = _hip.load_library()
    dtype, shape = _DTYPES.get(x.dtype), x.shape
    if dtype is None or len(shape) < 1 or shape[-1] == 0:
        raise ValueError("tokens must be float32, bfloat16 or float16 [..., C] with at least one channel")
    if x1 is not None and (x1.dtype != x.dtype or x1.shape[:-1] != shape[:-1] or x1.shape[-1] == 0):
        raise ValueError("the second source must have the first one's type and leading dimensions")
    c0, c1 = shape[-1], 0 if x1 is None else x1.shape[-1]
    c = c0 + c1
    if c > MAX_CHANNELS:
        raise ValueError("a token has at most %d channels" % MAX_CHANNELS)
    index = x.get_device()
    if index < 0:
        _elsewhere(x)
    x, rows, pitch0 = _rows(x)
    pitch1, x1_ptr = 0, None
    if x1 is not None:
        if x1.get_device() != index:
            _elsewhere(x1)
        x1, _, pitch1 = _rows(x1)
        x1_ptr = x1.data_ptr()
    pitch = (c + 15) // 16 * 16
    lead = shape[:-1]
    device = x.device
    codes = torch.empty(*lead, pitch, dtype=torch.int8, device=device)  # (sizes one by one: a tuple takes half a microsecond longer)
    scales = torch.empty(*lead, dtype=torch.float32, device=device) if lead else torch.empty((), dtype=torch.float32, device=device)
    if rows:
        _call(index, "rcv_i8_quantize_tokens", L.rcv_i8_quantize_tokens, x.data_ptr(), pitch0, c0, x1_ptr, pitch1, c1, dtype, rows,
                codes.data_ptr(), pitch, scales.data_ptr())
    return codes if pitch == c else codes[..., :c], scales


def _product(codes, scales, weight, bias, residual, relu, dtype, height, width):
    L = _hip.load_library()
    k, n, shape = weight.channels, weight.out_channels, codes.shape
    lead = shape[:-1]
    if codes.dtype != torch.int8 or len(shape) < 1 or shape[-1] != k:
        raise ValueError("codes must be int8 [..., %d] for this weight" % k)
    if scales.dtype != torch.float32 or scales.shape != lead:
        raise ValueError("scales must be float32 with one value per token")
    out_type = _DTYPES.get(dtype)
    if out_type is None:
        raise ValueError("output type must be torch.float32, torch.bfloat16 or torch.float16")
    index = codes.get_device()
    if index < 0:
        _elsewhere(codes)
    wcodes, wscales = weight.codes, weight.scales
    if scales.get_device() != index or wcodes.get_device() != index or wscales.get_device() != index:
        _elsewhere(next(t for t in (scales, wcodes, wscales) if t.get_device() != index))
    out = torch.empty(*lead, n, dtype=dtype, device=codes.device)
    bias_ptr = res_ptr = res_pitch = 0
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (n,):
            raise ValueError("bias must be float32 [%d]" % n)
        if bias.get_device() != index:
            _elsewhere(bias)
        bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    if residual is not None:
        if residual.dtype != dtype or residual.shape != out.shape:
            raise ValueError("residual must have the output's type and shape")
        if residual.get_device() != index:
            _elsewhere(residual)
        residual, _, res_pitch = _rows(residual)
        res_ptr = residual.data_ptr()
    codes, rows, pitch = _rows(codes, 16, 1 << 22)
    if rows == 0:
        return out
    ptr, need = codes.data_ptr(), (k + 15) // 16 * 16
    if rows == 1:  # (one row has no pitch of its own)
        pitch = need
    if pitch % 16 or ptr % 16 or (need != k and codes.untyped_storage().nbytes() - codes.storage_offset() < (rows - 1) * pitch + need):
        raise ValueError("token rows must start 16 bytes aligned and be readable up to a multiple of 16 channels: "
                         "take the codes as quantize_tokens lays them out")
    scales = scales.contiguous()
    args = _pack_args(_ARGS_BYTES, out_type, ptr, scales.data_ptr(), wcodes.data_ptr(), wscales.data_ptr(), bias_ptr, res_ptr,
                      out.data_ptr(), rows, pitch, res_pitch, n, k, n, height, width, 1 if relu else 0, 0)
    call, workspace_bytes = (L.rcv_i8_conv3x3, L.rcv_i8_conv3x3_workspace_bytes) if height else (L.rcv_i8_matmul, L.rcv_i8_matmul_workspace_bytes)
    nbytes = workspace_bytes(rows, k, n)
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=codes.device)
        _call(index, "int8 product", call, args, ws.data_ptr(), nbytes)
    else:
        _call(index, "int8 product", call, args, None, 0)
    return out


def matmul(codes, scales, weight, bias=None, residual=None, relu=False, dtype=torch.bfloat16):
    """act( (codes @ weight.T) * scales * weight scales + bias + residual ) -> [..., N] of `dtype`.

    codes int8 [..., K] and scales float32 [...] as quantize_tokens gives them, weight an Int8Weight of [N, K], bias float32 [N],
    residual [..., N] of `dtype`.  The integer sums are exact; float32 rounds their conversion, the product with the token's scale, the weight
    scale with the bias, and the residual, and the result is rounded to `dtype`.  relu keeps a NaN."""
    if weight.taps != 1:
        raise ValueError("matmul takes a weight packed from [N, K]; a 3x3 weight belongs to conv3x3")
    return _product(codes, scales, weight, bias, residual, relu, dtype, 0, 0)


def conv3x3(codes, scales, weight, bias=None, residual=None, relu=False, dtype=torch.bfloat16):
    """3x3 convolution with zero padding and stride 1 over tokens that form images: codes int8 [B, H, W, C], scales float32
    [B, H, W], weight an Int8Weight of [N, 3, 3, C] -> [B, H, W, N] of `dtype`.  Every input pixel enters under its own scale: integer
    sums over the channels of one tap, or over runs of them where a sum is divided, are exact, then converted and scaled; these are added
    in float32.  bias, residual, relu as in matmul."""
    if weight.taps != 9:
        raise ValueError("conv3x3 takes a weight packed from [N, 3, 3, C]")
    if codes.dim() != 4:
        raise ValueError("codes must be int8 [B, H, W, C]")
    return _product(codes, scales, weight, bias, residual, relu, dtype, codes.shape[1], codes.shape[2])
