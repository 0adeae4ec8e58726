"""Torch-facing launchers of the sm_100a Hyena kernels.

Each function validates shapes and dtypes on the host (ValueError, as the
reference's launchers do, mixers.py:479-509), builds the C-ABI argument structs
from tensor pointers and strides, and launches on the current CUDA stream.
Nothing here synchronises with the device, so all of it is CUDA-graph capturable
given fixed shapes (the HCL prefill workspace is the one allocation, made through
torch's caching allocator).

Kernel-side layouts:
  conv_state   (blocks, W0, 3H) bf16 view in vLLM's SD orientation (any strides)
  inner_state  FIR: (blocks, >=K-1, H) fp32 view; IIR: (blocks, H, >=16) fp32
  weights      LayerWeights, built once per layer by `layer_weights`
"""

from __future__ import annotations

import ctypes as C
import struct
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import DecodeArgs, LayerParams, PrefillArgs, StateView

BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _require(cond, msg):
    if not cond:
        raise ValueError(msg)


def _cuda(t, name):
    _require(t.is_cuda, f"{name} must be a CUDA tensor")


@dataclass
class LayerWeights:
    """Device tensors of one Hyena layer in the layout the kernels read.

    kind: "fir" or "iir". short_w (3H, 3) bf16 contiguous. FIR: inner_w_t (K, H)
    bf16 contiguous (the (H, K) taps transposed, so a warp reads consecutive
    channels of one tap). IIR: log_poles / residues (H, 16) fp32. D (H,) bf16 or None.
    """

    kind: str
    H: int
    K: int
    short_w: torch.Tensor
    inner_w_t: torch.Tensor | None = None
    log_poles: torch.Tensor | None = None
    residues: torch.Tensor | None = None
    D: torch.Tensor | None = None

    def params(self) -> LayerParams:
        p = LayerParams()
        p.kind = _lib.HYENA_KIND_FIR if self.kind == "fir" else _lib.HYENA_KIND_IIR
        p.H, p.K = self.H, self.K
        p.short_w = self.short_w.data_ptr()
        if self.kind == "fir":
            p.inner_w = self.inner_w_t.data_ptr()
            p.inner_w_stride_h = self.inner_w_t.stride(1)
            p.inner_w_stride_k = self.inner_w_t.stride(0)
        else:
            p.log_poles = self.log_poles.data_ptr()
            p.lp_stride_h, p.lp_stride_s = self.log_poles.stride()
            p.residues = self.residues.data_ptr()
            p.res_stride_h, p.res_stride_s = self.residues.stride()
        p.D = None if self.D is None else self.D.data_ptr()
        return p


def layer_weights(kind, short_filter, conv=None, D=None, log_poles=None, residues=None):
    """LayerWeights from checkpoint-layout parameters (mixers.py:805, 1247-1250,
    1323-1325): short_filter (3H,1,3), conv (H,1,K), D (H,), log_poles (H,S,1),
    residues (H,S)."""
    H = short_filter.shape[0] // 3
    short_w = short_filter.detach().reshape(3 * H, 3).to(BF16).contiguous()
    Dd = None if D is None else D.detach().to(BF16).contiguous()
    if kind == "fir":
        K = conv.shape[-1]
        inner = conv.detach().reshape(H, K).to(BF16).t().contiguous()
        return LayerWeights("fir", H, K, short_w, inner_w_t=inner, D=Dd)
    lp = log_poles.detach().reshape(H, -1).float().contiguous()
    res = residues.detach().reshape(H, -1).float().contiguous()
    return LayerWeights("iir", H, lp.shape[1], short_w, log_poles=lp, residues=res, D=Dd)


def state_view(t, cols_dim, chan_dim, cols=None) -> StateView:
    """A hyena_state_view over a (blocks, ...) tensor: `cols_dim` indexes window
    columns (or modes), `chan_dim` channels."""
    v = StateView()
    v.data = t.data_ptr()
    v.block_stride = t.stride(0)
    v.col_stride = t.stride(cols_dim)
    v.dim_stride = t.stride(chan_dim)
    v.cols = t.shape[cols_dim] if cols is None else cols
    v.num_blocks = t.shape[0]
    return v


def _check_states(w, conv_state, inner_state):
    _require(conv_state.dtype == BF16 and conv_state.dim() == 3 and conv_state.shape[2] == 3 * w.H,
             f"conv_state must be (blocks, W0, 3H) bf16, got {tuple(conv_state.shape)} {conv_state.dtype}")
    _require(conv_state.shape[1] >= 2, "conv_state needs at least 2 window columns")
    _require(inner_state.dtype == torch.float32 and inner_state.dim() == 3,
             "inner_state must be a 3-D fp32 tensor")
    if w.kind == "fir":
        _require(inner_state.shape[2] == w.H and inner_state.shape[1] >= w.K - 1,
                 f"FIR inner_state must be (blocks, >={w.K - 1}, H), got {tuple(inner_state.shape)}")
    else:
        _require(inner_state.shape[1] == w.H and inner_state.shape[2] >= w.K,
                 f"LI state must be (blocks, H, >={w.K}), got {tuple(inner_state.shape)}")


def _inner_view(w, inner_state):
    if w.kind == "fir":
        return state_view(inner_state, 1, 2, cols=w.K - 1)
    return state_view(inner_state, 2, 1, cols=w.K)


def _i32(t, name):
    if t.dtype != torch.int32:
        t = t.to(torch.int32)
    _cuda(t, name)
    return t


def prefill(w: LayerWeights, z, out, query_start_loc, has_initial_state, state_indices,
            conv_state, inner_state, error_flags=None):
    """Fused prefill core over packed rows: z (T, 3H) bf16 -> out (T, H) bf16.

    query_start_loc (n+1,) int32 segment offsets relative to z's first row;
    has_initial_state (n,) bool or None; state_indices (n,) int (any stride).
    """
    _require(z.dim() == 2 and z.shape[1] == 3 * w.H and z.dtype == BF16 and z.stride(1) == 1,
             f"z must be (T, 3H) bf16 with unit column stride, got {tuple(z.shape)}")
    _require(out.dim() == 2 and out.shape[1] == w.H and out.dtype == BF16 and out.stride(1) == 1,
             "out must be (T, H) bf16 with unit column stride")
    _require(out.shape[0] >= z.shape[0], "out has fewer rows than z")
    _cuda(z, "z")
    _check_states(w, conv_state, inner_state)
    n = state_indices.shape[0]
    _require(query_start_loc.numel() >= n + 1, "query_start_loc too short")
    qsl = _i32(query_start_loc[: n + 1].contiguous(), "query_start_loc")
    idx = _i32(state_indices, "state_indices")
    flags = None
    if has_initial_state is not None:
        flags = has_initial_state[:n]
        flags = (flags if flags.dtype == torch.bool else flags != 0).contiguous().view(torch.uint8)
    a = PrefillArgs()
    a.z, a.ldz = z.data_ptr(), z.stride(0)
    a.out, a.ldo = out.data_ptr(), out.stride(0)
    a.T = z.shape[0]
    a.num_segments = n
    a.query_start_loc = qsl.data_ptr()
    a.has_initial_state = None if flags is None else flags.data_ptr()
    a.state_indices = idx.data_ptr()
    a.state_indices_stride = idx.stride(0) if idx.dim() else 1
    a.conv_state = state_view(conv_state, 1, 2)
    a.inner_state = _inner_view(w, inner_state)
    a.error_flags = None if error_flags is None else error_flags.data_ptr()
    lib = _lib.load()
    p = w.params()
    ws_bytes = lib.hyena_prefill_workspace_size(C.byref(p), a.T, n)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=z.device) if ws_bytes else None
    # keep the temporaries alive until the launch returned
    _keep = (qsl, idx, flags, ws)
    _lib.check(lib.hyena_prefill(C.byref(p), C.byref(a), _ptr(ws), C.c_size_t(ws_bytes), _stream()),
               "hyena_prefill")
    del _keep
    return out


def decode(w: LayerWeights, z, out, conv_in_block, conv_out_block, in_slots, out_slots,
           conv_state, inner_state, token_start=None, accepted=None, zero_null_rows=False,
           skip_null_writes=True, null_block=0, error_flags=None):
    """Fused decode / speculative verify: z (tokens, 3H) -> out (tokens, H).

    conv_in_block / conv_out_block (B,) int; in_slots / out_slots (B, q) int
    (q = 1 for ordinary decode); token_start (B+1,) int or None (one token per
    request); accepted (B,) int (a count below 1 reads as 1) or None.
    """
    B = conv_in_block.shape[0]
    _require(z.dim() == 2 and z.shape[1] == 3 * w.H and z.dtype == BF16 and z.stride(1) == 1,
             "z must be (tokens, 3H) bf16")
    _require(out.dim() == 2 and out.shape[1] == w.H and out.dtype == BF16 and out.stride(1) == 1,
             "out must be (tokens, H) bf16")
    _check_states(w, conv_state, inner_state)
    _require(in_slots.dim() == 2 and out_slots.dim() == 2 and in_slots.shape[0] >= B
             and out_slots.shape[0] >= B, "slot tables must be (B, q)")
    q = out_slots.shape[1]
    _require(1 <= q <= 8, f"at most 8 positions per request, got {q}")
    if B == 0:
        return out
    cin = _i32(conv_in_block, "conv_in_block")
    cout = _i32(conv_out_block, "conv_out_block")
    if cin.dim() != 1 or cin.stride(0) < 1:
        cin = cin.contiguous().view(-1)
    if cout.dim() != 1 or cout.stride(0) < 1:
        cout = cout.contiguous().view(-1)
    ins = _i32(in_slots, "in_slots")
    outs = _i32(out_slots, "out_slots")
    ts = None if token_start is None else _i32(token_start[: B + 1], "token_start").contiguous()
    acc = None if accepted is None else _i32(accepted[:B], "accepted").contiguous()
    a = DecodeArgs()
    a.z, a.ldz = z.data_ptr(), z.stride(0)
    a.out, a.ldo = out.data_ptr(), out.stride(0)
    a.num_reqs, a.q = B, q
    a.token_start = None if ts is None else ts.data_ptr()
    a.accepted = None if acc is None else acc.data_ptr()
    a.conv_in_block, a.conv_out_block = cin.data_ptr(), cout.data_ptr()
    a.conv_in_stride, a.conv_out_stride = cin.stride(0), cout.stride(0)
    a.in_slots, a.in_stride0, a.in_stride1 = ins.data_ptr(), ins.stride(0), ins.stride(1)
    a.out_slots, a.out_stride0, a.out_stride1 = outs.data_ptr(), outs.stride(0), outs.stride(1)
    a.zero_null_rows = int(bool(zero_null_rows))
    a.skip_null_writes = int(bool(skip_null_writes))
    a.null_block = int(null_block)
    a.conv_state = state_view(conv_state, 1, 2)
    a.inner_state = _inner_view(w, inner_state)
    a.error_flags = None if error_flags is None else error_flags.data_ptr()
    lib = _lib.load()
    p = w.params()
    _keep = (cin, cout, ins, outs, ts, acc)
    _lib.check(lib.hyena_decode(C.byref(p), C.byref(a), _stream()), "hyena_decode")
    del _keep
    return out


def quant_e4m3(x, input_scale, out=None):
    """q = e4m3(clamp(x / sx, +-448)) (fp8_emul.py:76-78). x (M, K) bf16 -> (M, K) e4m3."""
    _require(x.dim() == 2 and x.dtype == BF16 and x.stride(1) == 1, "x must be (M, K) bf16")
    _require(input_scale.dtype == torch.float32 and input_scale.numel() == 1,
             "input_scale must be one fp32 element")
    M, K = x.shape
    if out is None:
        out = torch.empty(M, K, dtype=E4M3, device=x.device)
    lib = _lib.load()
    _lib.check(lib.hyena_quant_e4m3(_ptr(x), x.stride(0), _ptr(out), out.stride(0), M, K,
                                    _ptr(input_scale), _stream()), "hyena_quant_e4m3")
    return out


def gemm_fp8_emulated(a, w_t, scale_a, scale_b, out=None):
    """out (N, M) bf16 = Hopper fast-accumulation model of a (N, K) e4m3 . w_t (K, M)
    (bf16 holding E4M3 values), scaled by sa then sb (fp8_emul.py:45-88)."""
    _cuda(a, "a")
    _require(a.dtype == E4M3 and a.dim() == 2 and a.stride(1) == 1, "a must be (N, K) e4m3 rows")
    _require(w_t.dtype == BF16 and w_t.dim() == 2 and w_t.stride(1) == 1 and
             w_t.shape[0] == a.shape[1], "w_t must be (K, M) bf16 rows")
    N, K = a.shape
    M = w_t.shape[1]
    if out is None:
        out = torch.empty(N, M, dtype=BF16, device=a.device)
    lib = _lib.load()
    _lib.check(lib.hyena_gemm_fp8_emulated(_ptr(a), a.stride(0), _ptr(w_t), w_t.stride(0),
                                           _ptr(out), out.stride(0), N, M, K, _ptr(scale_a),
                                           _ptr(scale_b), _stream()), "hyena_gemm_fp8_emulated")
    return out


def fp8_linear_emulated(x, w_t, scales):
    """The FP8-surgery projection without FP8 hardware (mixers.py:701-705,
    fp8_emul_triton.py:181-191): q(x) with the static input scale scales[0],
    then the fast-accumulation model against w_t (K, M), times scales[0] * scales[1]."""
    _require(scales.dtype == torch.float32 and scales.numel() == 2, "scales must be 2 fp32")
    sx, sw = scales[0:1], scales[1:2]
    x2 = x.reshape(-1, x.shape[-1])
    q = quant_e4m3(x2.contiguous(), sx)
    return gemm_fp8_emulated(q, w_t, sx, sw).reshape(*x.shape[:-1], w_t.shape[1])


def rms_norm(x, weight, eps, residual=None, *, want_y=True, quant_scale=None, s_out=None):
    """Evo2RMSNorm of the decoder layer (model.py:47-76 Evo2RMSNorm.forward;
    triton_norm.py:127-156 rms_norm), one pass over the rows of x (M, H) bf16:

      s = x + residual (bf16), written to s_out (which may be x or residual:
          vLLM's in-place fused add-norm);
      y = weight * s / (||s||_2 * H^-0.5 + eps) with torch's bf16 roundings;
      q = e4m3(clamp(y / quant_scale, +-448)) when quant_scale is given.

    Returns (y or None, q or None).  want_y=False with quant_scale skips the
    bf16 output entirely (the in_proj input of a Hyena layer)."""
    _cuda(x, "x")
    _require(x.dim() == 2 and x.dtype == BF16 and x.stride(1) == 1, "x must be (M, H) bf16 rows")
    M, H = x.shape
    _require(weight.dtype == BF16 and weight.numel() == H and weight.is_contiguous(),
             "weight must be (H,) bf16")
    if residual is not None:
        _require(residual.shape == x.shape and residual.dtype == BF16 and residual.stride(1) == 1,
                 "residual must match x")
    if s_out is not None:
        _require(s_out.shape == x.shape and s_out.dtype == BF16 and s_out.stride(1) == 1,
                 "s_out must match x")
    if quant_scale is not None:
        _require(quant_scale.dtype == torch.float32 and quant_scale.numel() == 1,
                 "quant_scale must be one fp32 element")
    _require(want_y or quant_scale is not None or s_out is not None, "no output requested")
    y = torch.empty(M, H, dtype=BF16, device=x.device) if want_y else None
    q = torch.empty(M, H, dtype=E4M3, device=x.device) if quant_scale is not None else None
    lib = _lib.load()
    ld = lambda t: t.stride(0) if t is not None else 0  # noqa: E731
    _lib.check(lib.hyena_rms_norm(
        _ptr(x), x.stride(0), _ptr(residual), ld(residual), _ptr(weight), float(eps),
        _ptr(s_out), ld(s_out), _ptr(y), ld(y), _ptr(q), ld(q), _ptr(quant_scale), M, H,
        _stream()), "hyena_rms_norm")
    return y, q


def gemm_e4m3(a, b, scale_a, scale_b, out=None):
    """out (M, N) bf16 = (a (M,K) e4m3 . b (N,K) e4m3^T) * sa * sb (tcgen05)."""
    _require(a.dtype == E4M3 and b.dtype == E4M3, "e4m3 operands expected")
    _require(a.dim() == 2 and b.dim() == 2 and a.shape[1] == b.shape[1], "shape mismatch")
    _require(a.stride(1) == 1 and b.stride(1) == 1, "operands must be K-contiguous")
    M, K = a.shape
    N = b.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=BF16, device=a.device)
    lib = _lib.load()
    ws = _gemm_workspace(lib, M, N, K, True, a.device)
    _lib.check(lib.hyena_gemm_e4m3(_ptr(a), a.stride(0), _ptr(b), b.stride(0), _ptr(out),
                                   out.stride(0), M, N, K, _ptr(scale_a), _ptr(scale_b),
                                   _ptr(ws), C.c_size_t(0 if ws is None else ws.numel() * 4),
                                   _stream()), "hyena_gemm_e4m3")
    return out


def gemm_wait_timeouts(reset: bool = False) -> int:
    """Expired shared-memory barrier waits in the GEMMs on the current device
    since the last reset (hyena_gemm_wait_timeouts; synchronous).  Non-zero
    means some GEMM output was written from an incomplete tile."""
    n = C.c_int32(0)
    _lib.check(_lib.load().hyena_gemm_wait_timeouts(C.byref(n), int(bool(reset))),
               "hyena_gemm_wait_timeouts")
    return int(n.value)


def check_gemm_waits() -> None:
    """Raises RuntimeError when any GEMM wait expired on the current device."""
    n = gemm_wait_timeouts()
    if n:
        raise RuntimeError(f"{n} GEMM shared-memory barrier wait(s) expired: "
                           "GEMM outputs of this process are unreliable")


def set_gemm_max_ctas(n: int) -> None:
    """Caps the CTAs of the large-M GEMMs (0: one per SM) so that collectives
    running on another stream find free SMs (hyena_set_gemm_max_ctas)."""
    _lib.load().hyena_set_gemm_max_ctas(int(n))


def _stamp_view(stamps):
    """(base pointer, element stride) of a 1-D fp32 stamp view (one per block)."""
    _require(stamps.dim() == 1 and stamps.dtype == torch.float32, "stamps must be a 1-D fp32 view")
    return stamps.data_ptr(), stamps.stride(0)


def spec_accepted(slots, computed, stamps, num_spec, out=None, error_flags=None):
    """accepted (R,) int32 = clamp(computed - stamp(slots[:, 0]), 0, num_spec) + 1
    (hyena_spec_accepted; mixers.py:962-984).  slots (R,) or (R, S) int32."""
    lib = _lib.load()
    first = slots if slots.dim() == 1 else slots[:, 0]
    first = _i32(first, "slots")
    comp = _i32(computed[: first.shape[0]].contiguous(), "computed")
    R = first.shape[0]
    if out is None:
        out = torch.empty(R, dtype=torch.int32, device=first.device)
    base, stride = _stamp_view(stamps)
    _lib.check(lib.hyena_spec_accepted(first.data_ptr(), first.stride(0) if R else 1, R,
                                       comp.data_ptr(), base, stride, stamps.shape[0], int(num_spec),
                                       out.data_ptr(), _ptr(error_flags), _stream()),
               "hyena_spec_accepted")
    return out


def spec_record(out_slots, starts, computed, stamps, error_flags=None):
    """stamp(out_slots[r, p]) = computed[r] + p + 1 for the active positions p of
    each request (hyena_spec_record; mixers.py:1040-1062)."""
    lib = _lib.load()
    slots = _i32(out_slots if out_slots.dim() == 2 else out_slots[:, None], "out_slots")
    R, q = slots.shape
    st = _i32(starts[: R + 1].contiguous(), "starts")
    comp = _i32(computed[:R].contiguous(), "computed")
    base, stride = _stamp_view(stamps)
    _lib.check(lib.hyena_spec_record(slots.data_ptr(), slots.stride(0), slots.stride(1), R, q,
                                     st.data_ptr(), comp.data_ptr(), base, stride, stamps.shape[0],
                                     _ptr(error_flags), _stream()), "hyena_spec_record")


def spec_record_prefill(blocks, seq_lens, stamps, error_flags=None):
    """stamp(blocks[j]) = seq_lens[j] (hyena_spec_record_prefill;
    mixers.py:1070-1074).  blocks (n,) int (any stride), seq_lens (n,) int."""
    n = blocks.shape[0]
    if n == 0:
        return
    b = _i32(blocks, "blocks")
    lens = _i32(seq_lens[:n].contiguous(), "seq_lens")
    base, stride = _stamp_view(stamps)
    _lib.check(_lib.load().hyena_spec_record_prefill(
        b.data_ptr(), b.stride(0), n, lens.data_ptr(), base, stride, stamps.shape[0],
        _ptr(error_flags), _stream()), "hyena_spec_record_prefill")


def _block_slice(t):
    """A StateBlock over a paged (blocks, ...) tensor whose blocks are contiguous."""
    from ._lib import StateBlock

    inner = t[0] if t.shape[0] else t
    _require(inner.is_contiguous(), "state blocks must be contiguous within a block")
    sb = StateBlock()
    sb.data = t.data_ptr()
    sb.block_stride_bytes = t.stride(0) * t.element_size()
    sb.block_bytes = inner.numel() * t.element_size()
    return sb


def state_repair(dst_blocks, src_blocks, computed, has_init, stamps, states, error_flags=None):
    """Prefix-caching repair of resumed prefill rows (hyena_state_repair;
    mixers.py:1001-1037): where a row's destination block is not stamped with
    its computed-token count but its source block is, the source block's whole
    state (every tensor of `states`, each (blocks, ...)) is copied over the
    destination.  Returns the (n,) int32 decision (source block or -1)."""
    from ._lib import StateBlock

    n = dst_blocks.shape[0]
    take = torch.empty(max(n, 1), dtype=torch.int32, device=stamps.device)
    if n == 0:
        return take[:0]
    dst = _i32(dst_blocks, "dst_blocks")
    src = _i32(src_blocks[:n].contiguous(), "src_blocks")
    comp = _i32(computed[:n].contiguous(), "computed")
    init = has_init[:n]
    init = (init if init.dtype == torch.bool else init != 0).contiguous().view(torch.uint8)
    arr = (StateBlock * len(states))(*[_block_slice(t) for t in states])
    base, stride = _stamp_view(stamps)
    _lib.check(_lib.load().hyena_state_repair(
        n, dst.data_ptr(), dst.stride(0), src.data_ptr(), comp.data_ptr(), init.data_ptr(), base,
        stride, stamps.shape[0], arr, len(states), take.data_ptr(), _ptr(error_flags), _stream()),
        "hyena_state_repair")
    return take[:n]


def set_launch_chaining(enable: bool) -> None:
    """Programmatic dependent launch between this library's kernels on/off
    (hyena_set_launch_chaining; on by default)."""
    _lib.load().hyena_set_launch_chaining(int(bool(enable)))


def _gemm_workspace(lib, M, N, K, fp8, device):
    """Workspace the library asks for at this shape (none at present: small-M
    GEMMs reduce their K slices inside a thread-block cluster)."""
    n = lib.hyena_gemm_workspace_size(M, N, K, int(fp8))
    return torch.empty(n // 4, dtype=torch.float32, device=device) if n else None


def gemm_bf16(a, b, bias=None, out=None):
    """out (M, N) bf16 = a (M,K) bf16 . b (N,K) bf16^T [+ bias] (tcgen05)."""
    _require(a.dtype == BF16 and b.dtype == BF16, "bf16 operands expected")
    _require(a.dim() == 2 and b.dim() == 2 and a.shape[1] == b.shape[1], "shape mismatch")
    _require(a.stride(1) == 1 and b.stride(1) == 1, "operands must be K-contiguous")
    _require(bias is None or (bias.dtype == BF16 and bias.numel() == b.shape[0]), "bias must be (N,) bf16")
    M, K = a.shape
    N = b.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=BF16, device=a.device)
    lib = _lib.load()
    ws = _gemm_workspace(lib, M, N, K, False, a.device)
    _lib.check(lib.hyena_gemm_bf16(_ptr(a), a.stride(0), _ptr(b), b.stride(0), _ptr(out),
                                   out.stride(0), M, N, K, _ptr(bias), _ptr(ws),
                                   C.c_size_t(0 if ws is None else ws.numel() * 4), _stream()),
               "hyena_gemm_bf16")
    return out


# ---------------------------------------------------------------- attention cache, gated MLP
# These are called once a layer and decode step, so their host side counts: the
# argument structs are packed in one go (layouts as in include/hyena_b200.h,
# native alignment) and the stream is read without building a torch.cuda.Stream.
ACTIVATIONS = {"none": 0, "gelu": 1, "silu": 2}
PAGED_ATTENTION_REQUESTS = 2048  # requests and groups of one paged_attention call
_PAGED_KV = "PP6qPq5i"  # hyena_paged_kv
_KV_APPEND = struct.Struct("@PqqPqqPqqPqqPP3i" + _PAGED_KV + "dP")          # hyena_kv_append_args
_PAGED_ATTENTION = struct.Struct("@PqqPqqPPPP4if" + _PAGED_KV + "P")        # hyena_paged_attention_args


def _same_device(names, *tensors):
    """The index of the one CUDA device that the given tensors (None: absent) are
    on; refuses others, and tensors that need a gradient: these operators have no
    backward pass."""
    device = tensors[0].get_device()
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and (t.get_device() != device or (grad and t.requires_grad)):
            break
    else:
        if device >= 0:
            return device
    for name, t in zip(names.split(), tensors):
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
        if t.get_device() != device:
            raise ValueError(f"{name} is on {t.device}, not on {tensors[0].device}")
        if grad and t.requires_grad:
            raise ValueError(f"{name} requires grad: this operator has no backward pass "
                             "(call it under torch.no_grad())")


class _On:
    """`with _On(device) as stream:` makes the device current if it is not, and
    gives its current stream's handle."""

    __slots__ = ("device", "guard")

    def __init__(self, device):
        self.device, self.guard = device, None

    def __enter__(self):
        if torch._C._cuda_getDevice() != self.device:
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        return torch._C._cuda_getCurrentRawStream(self.device)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _rows3(t, name, heads, dim):
    """(tokens, token stride, head stride) of a (tokens, heads, dim) bf16 tensor."""
    shape = t.shape
    if len(shape) != 3 or t.dtype is not BF16:
        raise ValueError(f"{name} must be (tokens, heads, head_dim) bf16, got {tuple(shape)} {t.dtype}")
    n, h, d = shape
    if d != dim or (heads is not None and h != heads):
        raise ValueError(f"{name} must have {'' if heads is None else str(heads) + ' '}heads of {dim}, "
                         f"got {tuple(shape)}")
    a, b, c = t.stride()
    if c != 1:
        raise ValueError(f"{name} must have a unit last stride, got {t.stride()}")
    return n, a if n > 1 else 0, b if h > 1 else 0


def _ints(t, name, at_least):
    """A 1-D contiguous int32 tensor (converted if need be) of at least `at_least` elements."""
    shape = t.shape
    if len(shape) != 1 or shape[0] < at_least:
        raise ValueError(f"{name} must be 1-D with at least {at_least} elements, got {tuple(shape)}")
    if t.dtype is not torch.int32:
        if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
            raise ValueError(f"{name} must hold integers, got {t.dtype}")
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _paged_kv(k_cache, v_cache, page_table, requests):
    """The fields of hyena_paged_kv, and the page table they point to (None requests:
    as many as the table has rows)."""
    shape, k_strides, v_strides = k_cache.shape, k_cache.stride(), v_cache.stride()
    if (len(shape) != 4 or v_cache.shape != shape or k_cache.dtype is not BF16
            or v_cache.dtype is not BF16 or k_strides[3] != 1 or v_strides[3] != 1):
        for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
            if t.dim() != 4 or t.dtype is not BF16 or t.stride(3) != 1:
                raise ValueError(f"{name} must be (pages, page size, kv heads, head_dim) bf16 with unit "
                                 f"last stride, got {tuple(t.shape)} {t.dtype}")
        raise ValueError(f"k_cache {tuple(shape)} and v_cache {tuple(v_cache.shape)} differ")
    kp, kt, kh, _ = k_strides
    vp, vt, vh, _ = v_strides
    pages, size, heads, dim = shape
    if pages == 1:
        kp = vp = 0
    if heads == 1:
        kh = vh = 0
    table = page_table.shape
    if len(table) != 2 or (requests is not None and table[0] < requests) or page_table.is_floating_point():
        raise ValueError(f"page_table must be (>= {requests or 0} requests, pages) int, "
                         f"got {tuple(table)} {page_table.dtype}")
    row, one = page_table.stride()
    if page_table.dtype is not torch.int32 or (one != 1 and table[1] > 1):
        page_table = page_table.to(torch.int32).contiguous()
        row = page_table.stride(0)
    return (k_cache.data_ptr(), v_cache.data_ptr(), kp, kt, kh, vp, vt, vh, page_table.data_ptr(), row,
            table[1], pages, size, heads, dim), page_table


def _flags_ptr(error_flags):
    if error_flags is None:
        return 0
    _require(error_flags.dtype == torch.int32 and error_flags.numel() >= 1,
             "error_flags must be an int32 tensor")
    return error_flags.data_ptr()


def kv_append(q, k, v, positions, k_cache, v_cache, page_table, query_start_loc=None, *,
              rope_theta=10000.0, q_out=None, error_flags=None):
    """Rotary embedding of a step's queries and keys, with the rotated keys and the
    values written into the paged cache on the way (hyena_kv_append; the rotation
    of Evo2Attention, model.py:104-152).

    q (T, heads, D) or None; k, v (T, kv_heads, D): bf16, any token and head
    strides (views of the fused projection's output will do), D 64 or 128.
    positions (T,): the token's position, which is its rotation and its row of
    the cache; a negative one marks a token to leave alone.  Caches (pages, page
    size, kv_heads, D) with any strides, written in place; position p of request
    r lies in page page_table[r, p // page size], page size a multiple of 16.
    Request r owns the tokens [query_start_loc[r], query_start_loc[r + 1])
    (default: token r alone); tokens that no request owns are left alone.  A page
    outside the cache is not written and sets HYENA_FLAG_BLOCK_RANGE in
    error_flags.  No two tokens of a step may name the same row.

    Returns the rotated queries: q_out (may be q) or a new tensor; None for q None."""
    device = _same_device("k v positions k_cache v_cache page_table q query_start_loc q_out error_flags",
                          k, v, positions, k_cache, v_cache, page_table, q, query_start_loc, q_out,
                          error_flags)
    requests, starts = None, 0
    if query_start_loc is not None:
        query_start_loc = _ints(query_start_loc, "query_start_loc", 1)
        requests, starts = query_start_loc.shape[0] - 1, query_start_loc.data_ptr()
    kv, table = _paged_kv(k_cache, v_cache, page_table, requests)
    if requests is None:
        requests = table.shape[0]
    kv_heads, dim = kv[13], kv[14]
    T, k_token, k_head = _rows3(k, "k", kv_heads, dim)
    n, v_token, v_head = _rows3(v, "v", kv_heads, dim)
    if n != T:
        raise ValueError(f"v has {n} tokens, k {T}")
    heads = 0
    q_ptr = q_token = q_head = out_ptr = out_token = out_head = 0
    if q is not None:
        n, q_token, q_head = _rows3(q, "q", None, dim)
        if n != T:
            raise ValueError(f"q has {n} tokens, k {T}")
        heads = q.shape[1]
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            out_token, out_head = heads * dim, dim
        else:
            n, out_token, out_head = _rows3(q_out, "q_out", heads, dim)
            if n != T:
                raise ValueError(f"q_out has {n} tokens, q {T}")
        q_ptr, out_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    positions = _ints(positions, "positions", T)
    if T == 0 or requests == 0:
        return q_out
    args = _KV_APPEND.pack(q_ptr, q_token, q_head, out_ptr, out_token, out_head, k.data_ptr(), k_token,
                           k_head, v.data_ptr(), v_token, v_head, positions.data_ptr(), starts, T,
                           requests, heads, *kv, rope_theta, _flags_ptr(error_flags))
    with _On(device) as stream:
        rc = _lib.load().hyena_kv_append(args, stream)
    del table  # alive until the launch returned
    if rc:
        _lib.check(rc, "hyena_kv_append")
    return q_out


def paged_attention(q, k_cache, v_cache, page_table, seq_lens, query_start_loc=None, *,
                    shared_lens=None, group_start=None, scale=None, out=None, error_flags=None):
    """Causal attention of a step's queries over the paged cache, the leading keys
    that the requests of a group share read once for the group
    (hyena_paged_attention; Evo2Attention's softmax attention, model.py:104-152).

    q (T, heads, D) bf16, heads a multiple of kv_heads; caches and page_table as
    for kv_append.  seq_lens (B,): keys of request r, the step's own tokens
    (appended before) included; its n queries sit at the last n positions and see
    the keys up to their own.  Keys beyond the page table, and pages outside the
    cache, are left out and set HYENA_FLAG_BLOCK_RANGE in error_flags; a range of
    query_start_loc beyond T sets HYENA_FLAG_SEGMENT (its rows that exist keep
    their positions).  A request with seq_lens 0 (padding) gets zeros; rows that no
    request owns are left alone (uninitialised in a new `out`).
    shared_lens (G,): requests group_start[g] .. group_start[g + 1] - 1 (default:
    one group of all) name the same rows for their first shared_lens[g] keys; a
    run longer than what all of the group's queries see is cut, so the result
    never depends on it.  scale defaults to D ** -0.5.  B + G is at most 2048
    (PAGED_ATTENTION_REQUESTS).  out may be q itself.

    Two to four kernels (a plan, the shared runs of many rows, all other keys, and
    joining the pieces of split rows); lengths and tables are read on the device,
    so a captured graph serves growing contexts, and every call gives the same
    bits.  The workspace comes from torch's caching allocator.  Returns
    (T, heads, D) bf16."""
    device = _same_device("q k_cache v_cache page_table seq_lens query_start_loc shared_lens group_start "
                          "out error_flags", q, k_cache, v_cache, page_table, seq_lens, query_start_loc,
                          shared_lens, group_start, out, error_flags)
    seq_lens = _ints(seq_lens, "seq_lens", 0)
    requests = seq_lens.shape[0]
    kv, table = _paged_kv(k_cache, v_cache, page_table, requests)
    dim = kv[14]
    T, q_token, q_head = _rows3(q, "q", None, dim)
    heads = q.shape[1]
    starts = shared = group = groups = 0
    if query_start_loc is not None:
        query_start_loc = _ints(query_start_loc, "query_start_loc", requests + 1)
        starts = query_start_loc.data_ptr()
    if shared_lens is not None:
        shared_lens = _ints(shared_lens, "shared_lens", 1)
        groups, shared = shared_lens.shape[0], shared_lens.data_ptr()
        if group_start is not None:
            group_start = _ints(group_start, "group_start", groups + 1)
            group = group_start.data_ptr()
        elif groups > 1:
            raise ValueError("several groups need group_start")
    elif group_start is not None:
        raise ValueError("group_start without shared_lens")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        out_token, out_head = heads * dim, dim
    else:
        n, out_token, out_head = _rows3(out, "out", heads, dim)
        if n != T:
            raise ValueError(f"out has {n} tokens, q {T}")
    if T == 0 or requests == 0:
        return out
    args = _PAGED_ATTENTION.pack(
        q.data_ptr(), q_token, q_head, out.data_ptr(), out_token, out_head, seq_lens.data_ptr(), starts,
        shared, group, T, requests, groups, heads, dim ** -0.5 if scale is None else scale, *kv,
        _flags_ptr(error_flags))
    lib = _lib.load()
    with _On(device) as stream:
        n = lib.hyena_paged_attention_workspace_size(args)
        ws = q.new_empty(n // 2)  # bf16 elements
        rc = lib.hyena_paged_attention(args, ws.data_ptr(), n, stream)
    del table  # alive until the launch returned
    if rc:
        _lib.check(rc, "hyena_paged_attention")
    return out


def _matrix(t, name, cols=None):
    if t.dim() != 2 or t.dtype != BF16 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{name} must be a 2-D bf16 tensor with unit column stride, "
                         f"got {tuple(t.shape)} {t.dtype}")
    if cols is not None and t.shape[1] != cols:
        raise ValueError(f"{name} must have {cols} columns, got {tuple(t.shape)}")


def _ld(t):
    """Row stride; a one-row tensor may carry any: its length is what counts."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def gemm_gated_bf16(a, b1, b2, activation="none", out=None):
    """out (M, N) bf16 = act(a . b1^T) * (a . b2^T): a (M, K), b1 and b2 (N, K)
    bf16, activation "none", "gelu" (erf) or "silu", fp32 up to the one rounding
    (hyena_gemm_gated_bf16, tcgen05).  K % 64 == 0, N % 8 == 0."""
    device = _same_device("a b1 b2 out", a, b1, b2, out)
    _matrix(a, "a")
    M, K = a.shape
    _matrix(b1, "b1", K)
    _matrix(b2, "b2", K)
    N = b1.shape[0]
    _require(b2.shape[0] == N, f"b1 has {N} rows, b2 {b2.shape[0]}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if out is None:
        out = torch.empty(M, N, dtype=BF16, device=a.device)
    else:
        _matrix(out, "out", N)
        _require(out.shape[0] == M, f"out must have {M} rows, got {out.shape[0]}")
    with _On(device) as stream:
        rc = _lib.load().hyena_gemm_gated_bf16(a.data_ptr(), _ld(a), b1.data_ptr(), _ld(b1), b2.data_ptr(),
                                               _ld(b2), out.data_ptr(), _ld(out), M, N, K,
                                               ACTIVATIONS[activation], stream)
    if rc:
        _lib.check(rc, "hyena_gemm_gated_bf16")
    return out


def gated_mlp(x, w1, w2, w3, activation="none", out=None):
    """The gated feed-forward block of Evo2MLP (model.py:77-101):
    out (M, H) bf16 = (act(x . w1^T) * (x . w2^T)) . w3^T, x (M, H), w1 and w2
    (I, H), w3 (H_out, I) bf16; H and I multiples of 64.  Two launches: both
    projections with the activation and the product (gemm_gated_bf16, whose
    result is the one bf16 intermediate), then gemm_bf16."""
    device = _same_device("x w1 w2 w3 out", x, w1, w2, w3, out)
    _matrix(w1, "w1")
    _matrix(w3, "w3", w1.shape[0])
    _require(w1.shape[0] % 64 == 0, f"the inner width must be a multiple of 64, got {w1.shape[0]}")
    if out is not None:
        _matrix(out, "out", w3.shape[0])
        _require(out.shape[0] == x.shape[0], f"out must have {x.shape[0]} rows, got {out.shape[0]}")
    h = gemm_gated_bf16(x, w1, w2, activation)
    if out is None:
        out = torch.empty(h.shape[0], w3.shape[0], dtype=BF16, device=h.device)
    M, N = out.shape
    if M == 0 or N == 0:
        return out
    with _On(device) as stream:
        rc = _lib.load().hyena_gemm_bf16(h.data_ptr(), _ld(h), w3.data_ptr(), _ld(w3), out.data_ptr(), _ld(out),
                                         M, N, h.shape[1], None, None, 0, stream)
    if rc:
        _lib.check(rc, "hyena_gemm_bf16")
    return out
