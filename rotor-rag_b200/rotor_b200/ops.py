"""Tensor-level wrappers over the C ABI.  torch tensors are buffers only: every
function here allocates its outputs with torch and hands raw pointers to
librotor_b200.so on the current CUDA stream."""
from __future__ import annotations

import struct

import numpy as np

from . import abi
from .abi import lib, ptr, check


def _torch():
    return abi.require_cuda()


def to_device(a, dtype=None):
    """numpy array / tensor -> contiguous CUDA tensor."""
    torch = _torch()
    if isinstance(a, np.ndarray):
        a = torch.from_numpy(np.ascontiguousarray(a))
    elif a.dtype is dtype and a.is_contiguous() and a.get_device() == torch.cuda.current_device():
        return a             # (what the three conversions below come to; each costs about a microsecond)
    if dtype is not None:
        a = a.to(dtype)
    return a.contiguous().cuda()


# ------------------------------------------------------------------ format
def encode(w):
    torch = _torch()
    w = to_device(w, torch.int8).reshape(-1)
    plus = torch.empty(w.numel(), dtype=torch.uint8, device="cuda")
    minus = torch.empty_like(plus)
    check(lib.rotor_b200_encode(ptr(w), w.numel(), ptr(plus), ptr(minus), abi.stream()), "encode")
    return plus, minus


def decode(plus, minus):
    torch = _torch()
    plus, minus = to_device(plus, torch.uint8).reshape(-1), to_device(minus, torch.uint8).reshape(-1)
    w = torch.empty(plus.numel(), dtype=torch.int8, device="cuda")
    check(lib.rotor_b200_decode(ptr(plus), ptr(minus), plus.numel(), ptr(w), abi.stream()), "decode")
    return w


def pack(plus, minus):
    torch = _torch()
    plus, minus = to_device(plus, torch.uint8).reshape(-1), to_device(minus, torch.uint8).reshape(-1)
    n = plus.numel()
    packed = torch.empty(n // 4, dtype=torch.uint8, device="cuda")
    check(lib.rotor_b200_pack(ptr(plus), ptr(minus), n, ptr(packed), abi.stream()), "pack")
    return packed


def unpack(packed, n):
    torch = _torch()
    packed = to_device(packed, torch.uint8).reshape(-1)
    if packed.numel() * 4 < n:
        raise ValueError("packed array shorter than n rotors")
    plus = torch.empty(n, dtype=torch.uint8, device="cuda")
    minus = torch.empty_like(plus)
    check(lib.rotor_b200_unpack(ptr(packed), n, ptr(plus), ptr(minus), abi.stream()), "unpack")
    return plus, minus


def packed_to_planes(packed, cols=None):
    torch = _torch()
    packed = to_device(packed, torch.uint8)
    rows, nb = packed.shape
    cols = nb * 4 if cols is None else cols
    plus = torch.empty((rows, (cols + 7) // 8), dtype=torch.uint8, device="cuda")
    minus = torch.empty_like(plus)
    check(lib.rotor_b200_packed_to_planes(ptr(packed), rows, cols, ptr(plus), ptr(minus), abi.stream()),
          "packed_to_planes")
    return plus, minus


def planes_to_int8(plus, minus, rows, cols):
    torch = _torch()
    plus, minus = to_device(plus, torch.uint8), to_device(minus, torch.uint8)
    w = torch.empty((rows, cols), dtype=torch.int8, device="cuda")
    check(lib.rotor_b200_planes_to_int8(ptr(plus), ptr(minus), rows, cols, ptr(w), abi.stream()), "planes_to_int8")
    return w


# ------------------------------------------------------------------ tiles
def packed_to_tiles(packed, out, inn):
    torch = _torch()
    packed = to_device(packed, torch.uint8)
    if tuple(packed.shape) != (out, (inn + 3) // 4):
        raise ValueError(f"packed shape {tuple(packed.shape)} does not match [{out}, {(inn + 3) // 4}]")
    tiles = torch.empty(lib.rotor_b200_tiles_bytes(out, inn), dtype=torch.uint8, device="cuda")
    check(lib.rotor_b200_packed_to_tiles(ptr(packed), out, inn, ptr(tiles), abi.stream()), "packed_to_tiles")
    return tiles


def int8_to_tiles(w):
    torch = _torch()
    w = to_device(w, torch.int8)
    out, inn = w.shape
    tiles = torch.empty(lib.rotor_b200_tiles_bytes(out, inn), dtype=torch.uint8, device="cuda")
    check(lib.rotor_b200_int8_to_tiles(ptr(w), out, inn, ptr(tiles), abi.stream()), "int8_to_tiles")
    return tiles


def tiles_to_int8(tiles, out, inn):
    torch = _torch()
    w = torch.empty((out, inn), dtype=torch.int8, device="cuda")
    check(lib.rotor_b200_tiles_to_int8(ptr(tiles), out, inn, ptr(w), abi.stream()), "tiles_to_int8")
    return w


# ------------------------------------------------------------------ quantiser / BitLinear
def quantize_rows(x, terms=1):
    """x float32 [M, K] (CUDA) -> xq int8 [M*terms, K128], sx float32 [M*terms], xsum int32 [M*terms]."""
    torch = _torch()
    x = to_device(x, torch.float32)
    m, k = x.shape
    kpad = lib.rotor_b200_in_padded(k)
    xq = torch.empty((m * terms, kpad), dtype=torch.int8, device="cuda")
    sx = torch.empty(m * terms, dtype=torch.float32, device="cuda")
    xsum = torch.empty(m * terms, dtype=torch.int32, device="cuda")
    check(lib.rotor_b200_quantize_rows(ptr(x), m, k, terms, ptr(xq), ptr(sx), ptr(xsum), abi.stream()),
          "quantize_rows")
    return xq, sx, xsum


def bitlinear_acc(tiles, out, inn, xq, xsum, variant=abi.VARIANT_AUTO):
    """Exact int32 accumulators [ncols, out]."""
    torch = _torch()
    ncols = xq.shape[0]
    acc = torch.empty((ncols, out), dtype=torch.int32, device="cuda")
    check(lib.rotor_b200_bitlinear_acc(ptr(tiles), out, inn, ptr(xq), ptr(xsum), ncols, ptr(acc), variant,
                                       abi.stream()), "bitlinear_acc")
    return acc


def bitlinear_forward(tiles, out, inn, x, terms, wscale=1.0, wscale_vec=None, variant=abi.VARIANT_AUTO,
                      workspace=None):
    """y float32 [M, out] = BitLinear(x float32 [M, in])."""
    torch = _torch()
    x = to_device(x, torch.float32)
    need = lib.rotor_b200_bitlinear_workspace_bytes(out, inn, x.shape[0], terms)
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
    return bitlinear_into(tiles, out, inn, x, terms, float(wscale), ptr(wscale_vec), variant, workspace)


def bitlinear_into(tiles, out, inn, x, terms, wscale, wscale_vec, variant, workspace):
    """The call itself: x on the current device, float32 and contiguous, a workspace that is large enough."""
    m = x.shape[0]
    y = x.new_empty((m, out))
    status = lib.rotor_b200_bitlinear_forward(ptr(tiles), out, inn, x.data_ptr(), m, terms, wscale, wscale_vec, y.data_ptr(),
                                              workspace.data_ptr(), workspace.numel(), variant, abi.stream())
    if status:
        check(status, "bitlinear_forward")
    return y


def sample(logits, mode, top_k=50, top_p=0.9, temperature=1.0, seed=0, counter=0):
    """One token per row of CUDA float32 logits [rows, vocab]; mode 0 top-k, 1 top-p.  Returns a CUDA int64 [rows]."""
    torch = _torch()
    rows, vocab = logits.shape
    out = torch.empty(rows, dtype=torch.int64, device="cuda")
    abi.check(abi.lib.rotor_b200_sample(abi.ptr(logits), rows, vocab, int(mode), int(top_k), float(top_p),
                                        float(temperature), int(seed) & (2 ** 64 - 1), int(counter) & (2 ** 64 - 1),
                                        abi.ptr(out), abi.stream()), "sample")
    return out


# ------------------------------------------------------------------ beam search
# (calls of one token or one request are bound by the host: what Python does in them is kept short)
_CODES = {}


def type_code(dtype):
    """The C ABI's number of a floating type that the generation operators take."""
    if not _CODES:
        torch = _torch()
        _CODES.update({torch.float32: abi.F32, torch.bfloat16: abi.BF16, torch.float16: abi.F16})
    code = _CODES.get(dtype)
    if code is None:
        raise ValueError(f"{dtype} is not one of float32, bfloat16, float16")
    return code


def on_device(name, t, device, dim=None, dtype=None):
    """The tensor is on that CUDA device, of that many dimensions and that type."""
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not on the current CUDA device")
    if dim is not None and t.dim() != dim:
        raise ValueError(f"{name} of shape {tuple(t.shape)} where {dim} dimensions are expected")
    if dtype is not None and t.dtype is not dtype:
        raise ValueError(f"{name} is {t.dtype}, expected {dtype}")


def beam_select(logits, scores, count, ended=None, pad=0):
    """The ``count`` best continuations of every group of beams, best first: scores float32, beams and tokens int64, each
    [groups, count] on the device.

    ``logits`` [groups, width, vocab] (float32, bfloat16 or float16, tokens of a row side by side) after the beams, whose scores so
    far are ``scores`` float32 [groups, width]; a candidate is worth its beam's score plus the log-softmax of its logit.  Among equal
    ones the lower beam, then the lower token comes first; candidates of different beams that lie closer than the float32 sum of a
    row's exponentials is known (2e-7 of a score as measured) come in either order, the same one at every call.  ``ended`` bool [groups, width]: such a beam offers itself alone, as
    token ``pad`` with its score unchanged.  Logits of -inf or NaN, rows that hold +inf and beams whose score is not finite offer
    nothing; places that no candidate is left for hold -inf and the lowest unused (beam, token).  Up to 32 beams and 64 continuations."""
    device, stream = abi.device_and_stream()
    torch = abi._torch
    on_device("logits", logits, device, 3)
    on_device("scores", scores, device, 2, torch.float32)
    groups, width, vocab = logits.shape
    group_stride, beam_stride, side_by_side = logits.stride()
    code, count = type_code(logits.dtype), int(count)
    if tuple(scores.shape) != (groups, width):
        raise ValueError(f"scores of shape {tuple(scores.shape)}, expected {(groups, width)}")
    if side_by_side != 1 and vocab > 1:
        raise ValueError("the logits of a row have to lie side by side")
    if not (1 <= width <= 32 and 1 <= count <= 64 and count <= width * vocab < 2 ** 31 and vocab <= 2 ** 30):
        raise ValueError(f"{count} of {width} x {vocab} candidates: up to 32 beams and 64 continuations, not more than there are")
    if ended is not None:
        on_device("ended", ended, device, 2, torch.bool)
        if tuple(ended.shape) != (groups, width):
            raise ValueError(f"ended of shape {tuple(ended.shape)}, expected {(groups, width)}")
        if not 0 <= pad < vocab:
            raise ValueError(f"padding token {pad} of {vocab}")
        ended = ended.contiguous()
    if not scores.is_contiguous():
        scores = scores.contiguous()
    shape = (groups, count)
    best = scores.new_empty(shape)
    beams = scores.new_empty(shape, dtype=torch.int64)
    tokens = torch.empty_like(beams)
    if groups == 0:
        return best, beams, tokens
    if groups * width > 65535:
        raise ValueError(f"{groups} groups of {width} beams: up to 65535 beams in a call")
    call = (logits.data_ptr(), code, group_stride, beam_stride, scores.data_ptr(), None if ended is None else ended.data_ptr(), groups, width,
            vocab, count, int(pad), best.data_ptr(), beams.data_ptr(), tokens.data_ptr())
    status = lib.rotor_b200_beam_select(*call, None, 0, stream)
    if status == abi.ERR_WORKSPACE:      # (nothing has been launched; few logits need none)
        need = lib.rotor_b200_beam_select_workspace_bytes(code, groups, width, vocab, count)
        workspace = scores.new_empty(need, dtype=torch.uint8)
        status = lib.rotor_b200_beam_select(*call, workspace.data_ptr(), need, stream)
    if status:
        check(status, "beam_select")
    return best, beams, tokens


_STATE = struct.Struct("PNNNi4x")      # rotor_b200_state


def reorder_states(states, beams, length=None):
    """Row ``b * width + w`` of every state becomes what row ``b * width + beams[b, w]`` was, in place and in one launch: after
    ``beam_select`` the caches and histories follow the beams they continue.

    ``states``: tensors [groups * width, ...] whose rows are contiguous, or pairs (tensor, axis) of which the first ``length`` positions
    along that axis move; their memory may not overlap.  ``beams`` int64 [groups, width], up to 32 wide; rows whose beam is their own, or none of the group, stay."""
    device, stream = abi.device_and_stream()
    on_device("beams", beams, device, 2, abi._torch.int64)
    groups, width = beams.shape
    rows = groups * width
    if width > 32:
        raise ValueError(f"{width} beams: up to 32")
    described, addresses = [], set()
    for s in states:
        t, axis = s if isinstance(s, tuple) else (s, None)
        if length is None:
            axis = None
        shape = t.shape
        if t.get_device() != device:
            raise ValueError(f"a state is on {t.device}, not on the current CUDA device")
        if not shape or shape[0] != rows:
            raise ValueError(f"a state of shape {tuple(shape)} for {groups} x {width} beams")
        if axis is not None:
            if not 1 <= axis < len(shape):
                raise ValueError(f"positions along axis {axis} of a state of {len(shape)} dimensions")
            if not 0 <= length <= shape[axis]:
                raise ValueError(f"{length} positions of a state that holds {shape[axis]}")
        n = t.numel()
        if n == 0:
            continue
        size = t.element_size()
        row = row_stride = n // rows * size
        if not t.is_contiguous():
            row_stride = t.stride(0) * size
            if not t[0].is_contiguous() or (rows > 1 and row_stride < row):
                raise ValueError(f"a state's rows have to be contiguous and apart; got shape {tuple(shape)}, strides {t.stride()}")
        address = t.data_ptr()
        if address in addresses:
            raise ValueError("the same state twice")
        addresses.add(address)
        if axis is None:
            described.append(_STATE.pack(address, row_stride, row, row, 1))
        elif length:
            segments = 1          # (pieces of a row: what lies in front of the axis)
            for k in range(1, axis):
                segments *= shape[k]
            piece = row // segments
            described.append(_STATE.pack(address, row_stride, piece, piece // shape[axis] * length, segments))
    if not described:
        return
    beams = beams.contiguous()
    status = lib.rotor_b200_reorder_states(b"".join(described), len(described), beams.data_ptr(), groups, width, stream)
    if status:
        check(status, "reorder_states")
