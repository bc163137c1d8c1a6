"""Mamba-2 mixer with every stage between the two projections on the HIP kernels of this package; the module-level
interface of linquant/quantized_mamba2.py:36-378 (constructor keywords, calibrated buffers, forward arguments, the
prefill-only restriction and its error messages).

Pipeline of ``forward`` (linquant/quantized_mamba2.py:205-378):
  1. activation quantizer -> in_proj -> split z0, x0, z, xBC, dt
  2. causal conv1d + SiLU on xBC (mask applied before and after)
  3. split + optional D_qk rescale + Kronecker-Hadamard rotation + INT8 of B, C (x stays an fp16 view); key side: fp B rotated
  4. INT8 SSD (cumsum, chunk state, fixed-point state passing, C.B^T, chunk scan) -> fp16 y
  5. gated RMSNorm(y, z) and 6. Hadamard + INT8 of the out_proj input -- one launch when the norm is this package's
     RMSNormGated and d_mlp = 0 -- then out_proj and 7. the output compensation

The two projections are not part of this package: ``Int8InputLinear`` stands in for the W4A8 Marlin linear with the
same ``input_scale`` / ``forward_int8(x_i8, scale)`` surface and an fp16 GEMM from torch behind it, so the mixer runs
end to end on a ROCm build and the stage names below can be re-bound for per-stage timing exactly like
bench/mamba2_components.py:56-77 of the reference does.  ``linear=W8A8Linear`` puts this package's INT8 product in their place.

``forward`` is the reference's prefill and keeps nothing.  ``prefill`` and ``step`` serve: they carry each sequence's last
convolution inputs and its fp32 state from call to call in the slots of a ``Mamba2State``, for prompts of any lengths (whole, in
parts, packed) and for one token of each sequence, with the convolution and the scan in 16 bits between the same two projections.
``Mamba2Block`` puts the residual stream and its norm around a mixer.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn

from linquant_amd import _lib
from linquant_amd.hadamard_utils import qhad_transform
from linquant_amd.kernels.hadamard import kronecker_hadamard_fwd  # noqa: F401  (kept re-bindable like the reference's import)
from linquant_amd.kernels.mamba2.causal_conv1d import causal_conv1d_fn
from linquant_amd.kernels.mamba2.conv1d_state import conv1d_prompt, conv1d_step
from linquant_amd.kernels.mamba2.fused_split_rotate_xBC import fused_split_rotate_quant_xBC, prepare_dqk
from linquant_amd.kernels.mamba2.ssd_combined import _quant_mamba_chunk_scan_combined_fwd
from linquant_amd.kernels.mamba2.ssm import ssm_prompt, ssm_step
from linquant_amd.norm import RMSNormGated, residual_rmsnorm, rmsnorm_gated_qhad
from linquant_amd.w4a8_linear import _fused_fp16_to_int8


def _apply_mask(hidden_states, attention_mask):
    """Zero the padded positions (linquant/quantized_mamba2.py:28-33)."""
    if attention_mask is not None and attention_mask.shape[1] > 1:
        hidden_states = (hidden_states * attention_mask[:, :, None]).to(hidden_states.dtype)
    return hidden_states


class Int8InputLinear(nn.Module):
    """Stand-in for W4A8B16O16Linear (linquant/w4a8_linear.py): INT8 activations on a per-tensor static scale, fp16
    output.  The weight stays fp16 and the product is torch's fp16 GEMM of the dequantized activations."""

    def __init__(self, weight: torch.Tensor, input_scale: torch.Tensor, bias: torch.Tensor | None = None):
        super().__init__()
        self.register_buffer("weight", weight.detach().to(torch.float16).contiguous())
        self.register_buffer("input_scale", torch.as_tensor(input_scale, dtype=torch.float32).reshape(()).clone())
        self.register_buffer("bias", None if bias is None else bias.detach().to(torch.float16))

    @classmethod
    def from_fp16(cls, linear: nn.Linear, input_scale):
        return cls(linear.weight, input_scale, linear.bias)

    def forward_int8(self, x_i8: torch.Tensor, scale) -> torch.Tensor:
        s = scale.to(device=x_i8.device, dtype=torch.float32) if isinstance(scale, torch.Tensor) else float(scale)
        if isinstance(s, torch.Tensor) and s.numel() != 1:  # one for each row
            s = s.reshape(*x_i8.shape[:-1], 1)
        return torch.nn.functional.linear((x_i8.to(torch.float32) * s).to(torch.float16), self.weight, self.bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x2 = x.reshape(-1, x.shape[-1])
        q = _fused_fp16_to_int8(x2, self.input_scale.to(x.device))
        return self.forward_int8(q.view(x.shape), self.input_scale)


class Mamba2State(NamedTuple):
    """What sequences leave for their next tokens, a slot for each; zeros are the state of a sequence without tokens."""

    conv: torch.Tensor  # (slots, d_conv - 1, conv_dim) fp16: the last inputs of the convolution, oldest first
    ssm: torch.Tensor   # (slots, nheads, headdim, d_state) fp32


class _AsLaidOut:
    """The tensors that something was made of, to tell whether they still are the same: the objects, where their entries lie and how often
    they were written to.  (A copy or a loaded pickle of it, which has the copied module's tensors, marks them anew.)"""

    def __init__(self, *tensors):
        self.tensors = tensors
        # (a tensor of inference mode does not count its writes)
        self.marks = [(t, t.data_ptr(), not t.is_inference() and t._version) if isinstance(t, torch.Tensor) else (t, None, None) for t in tensors]

    def __reduce__(self):
        return _AsLaidOut, self.tensors

    def holds(self, tensors):
        for t, (was, at, writes) in zip(tensors, self.marks):
            if t is not was or (at is not None and (t.data_ptr() != at or (writes is not False and t._version != writes))):
                return False
        return True


class QuantizedMamba2(nn.Module):
    """Calibrated buffers attached after construction, as in the reference: B_scale/B_inv_scale, C_scale/C_inv_scale
    (G,), A_log_scale, D_scale (scalars), alpha_hp (H, P), bscale_g (G,), static_state_scale (H, P), static_cb_scale
    (G,), r_signs (G, N) or None, comp_out (d_model) or absent, dqk_b/dqk_c (G*N) or absent; key side additionally
    ``keyside = True``, x_quant_scale_hp (H, P) and b_gate_scale (1, 1, H, N)."""

    def __init__(self, *, d_model, d_ssm, nheads, headdim, d_state, ngroups, d_conv, chunk_size, in_proj, out_proj,
                 conv1d, norm, A_log, D, dt_bias, dt_limit=(0.0, float("inf")), layer_idx=None):
        super().__init__()
        self.d_model, self.d_ssm, self.nheads, self.headdim = d_model, d_ssm, nheads, headdim
        self.d_state, self.ngroups, self.d_conv, self.chunk_size = d_state, ngroups, d_conv, chunk_size
        self.dt_limit, self.layer_idx = tuple(dt_limit), layer_idx
        self.conv_dim = d_ssm + 2 * ngroups * d_state
        self.register_buffer("_one", torch.tensor(1.0, dtype=torch.float32))
        self.in_proj, self.out_proj, self.conv1d, self.norm = in_proj, out_proj, conv1d, norm
        self.register_buffer("A_log", A_log)   # INT8, dequantized in the cumsum kernel with A_log_scale
        self.D = D                             # INT8, dequantized in the scan with D_scale
        self.dt_bias = dt_bias
        self._serving = None

    @classmethod
    def from_fp16(cls, original_mixer, scales, r_signs, linear=Int8InputLinear):
        """Same contract as linquant/quantized_mamba2.py:105-203: ``original_mixer`` is any module with the Mamba2
        attributes (mamba-ssm or HF names), ``scales`` holds B/C/A_log/D scales and the two projection input scales.
        ``linear``: what the projections become (``Int8InputLinear`` or ``W8A8Linear``); an ``in_proj_input_scale`` of None
        lets a ``W8A8Linear`` quantize each row of the mixer's input on a scale of its own."""

        def pick(*names):
            for n in names:
                v = getattr(original_mixer, n, None)
                if v is not None:
                    return v
            return None

        nheads, headdim = pick("nheads", "num_heads"), pick("headdim", "head_dim")
        dt_limit = pick("dt_limit", "time_step_limit") or (0.0, float("inf"))
        q_A_log = torch.clamp(torch.round(original_mixer.A_log.float() * scales["A_log_inv_scale"]), -127, 127).to(torch.int8)
        q_D = torch.clamp(torch.round(original_mixer.D.float() * scales["D_inv_scale"]), -127, 127).to(torch.int8)
        module = cls(
            d_model=pick("d_model", "hidden_size"), d_ssm=nheads * headdim, nheads=nheads, headdim=headdim,
            d_state=pick("d_state", "ssm_state_size"), ngroups=pick("ngroups", "n_groups"),
            d_conv=pick("d_conv", "conv_kernel_size"), chunk_size=original_mixer.chunk_size,
            in_proj=linear.from_fp16(original_mixer.in_proj, scales["in_proj_input_scale"]),
            out_proj=linear.from_fp16(original_mixer.out_proj, scales["out_proj_input_scale"]),
            conv1d=original_mixer.conv1d, norm=original_mixer.norm, A_log=q_A_log, D=q_D,
            dt_bias=original_mixer.dt_bias, dt_limit=tuple(dt_limit), layer_idx=getattr(original_mixer, "layer_idx", None))
        module.register_buffer("r_signs", r_signs)
        for name in ("B_scale", "B_inv_scale", "C_scale", "C_inv_scale", "A_log_scale", "D_scale"):
            module.register_buffer(name, scales[name])
        return module

    @torch.no_grad()
    def forward(self, hidden_states, attention_mask=None, past_key_values=None, use_cache=False,
                output_attentions=False, **kwargs):
        if past_key_values is not None or kwargs.get("inference_params") is not None:
            raise NotImplementedError(
                "QuantizedMamba2 is prefill-only: cached/stateful decoding (past_key_values, inference_params) is not "
                "implemented; the conv history and the SSM state are not carried between calls")
        debug = kwargs.get("_debug")
        if hidden_states.dtype == torch.bfloat16:
            hidden_states = hidden_states.to(torch.float16)

        # 1. in_proj on INT8 activations (rint(x / s) clamped to [-128, 127])
        h_i8, projected = self._in_project(hidden_states)
        z0, x0, z, xBC, dt = self._split(projected)

        # 2. causal conv1d + SiLU
        xBC = _apply_mask(xBC, attention_mask)
        xBC = causal_conv1d_fn(x=xBC.transpose(1, 2), weight=self.conv1d.weight.reshape(self.conv_dim, -1),
                               bias=self.conv1d.bias, activation="silu").transpose(1, 2)
        xBC = _apply_mask(xBC, attention_mask)

        # 3. split, rotate and quantize B / C; x stays an fp16 view of xBC
        dqk_b, dqk_c = getattr(self, "dqk_b", None), getattr(self, "dqk_c", None)
        if dqk_b is not None:
            if getattr(self, "_dqk_prepared", None) is None:
                self._dqk_prepared = (prepare_dqk(dqk_b), prepare_dqk(dqk_c))
            dqk_b, dqk_c = self._dqk_prepared
        r_signs = getattr(self, "r_signs", None)
        keyside = getattr(self, "keyside", False)
        keyside_kwargs = {}
        if keyside:  # the fp B of the key-side chunk state carries D_qk and the rotation q_B was quantized under: the
            # prologue kernel stores it next to the codes (one launch instead of the reference's two), with its per-token
            # maxima, which the chunk state stage would otherwise compute in a pass of its own
            x_fp, q_B, q_C, b_fp, b_rowmax = fused_split_rotate_quant_xBC(
                xBC, r_signs, self.nheads, self.ngroups, self.d_state, self.headdim, self.B_inv_scale, self.C_inv_scale,
                dqk_b=dqk_b, dqk_c=dqk_c, return_b_fp=True, return_b_rowmax=True)
            keyside_kwargs = dict(keyside=True, x_scale_hp=self.x_quant_scale_hp, b_fp=b_fp, b_gate_scale=self.b_gate_scale,
                                  b_rowmax=b_rowmax)
        else:
            x_fp, q_B, q_C = fused_split_rotate_quant_xBC(xBC, r_signs, self.nheads, self.ngroups, self.d_state,
                                                          self.headdim, self.B_inv_scale, self.C_inv_scale,
                                                          dqk_b=dqk_b, dqk_c=dqk_c)

        # 4. INT8 SSD
        missing = [n for n in ("alpha_hp", "bscale_g", "static_state_scale", "static_cb_scale") if not hasattr(self, n)]
        if missing:
            raise RuntimeError(f"QuantizedMamba2 is not calibrated: missing buffers {missing} "
                               "(from_fp16 builds the module; the calibration step must attach these before inference)")
        dt_limit_kwargs = {} if self.dt_limit == (0.0, float("inf")) else {"dt_limit": self.dt_limit}
        y, _ = _quant_mamba_chunk_scan_combined_fwd(
            x_fp=x_fp, q_dt=dt, dt_scale=self._one.to(device=dt.device), q_A_log=self.A_log, A_log_scale=self.A_log_scale,
            q_B=q_B, B_scale=self.B_scale, q_C=q_C, C_scale=self.C_scale, chunk_size=self.chunk_size, q_D=self.D,
            D_scale=self.D_scale, dt_bias=self.dt_bias, dt_softplus=True, alpha_hp=self.alpha_hp, bscale_g=self.bscale_g,
            static_state_scale=self.static_state_scale, static_cb_scale=self.static_cb_scale, **keyside_kwargs,
            **dt_limit_kwargs)
        y = y.reshape(y.shape[0], y.shape[1], self.d_ssm)

        # 5 - 7. gated RMSNorm, Hadamard + INT8 of the out_proj input, out_proj, output compensation
        out, normed, y_i8 = self._finish(y, z, z0, x0)
        if debug is not None:
            debug.update(h_i8=h_i8, projected=projected, xBC=xBC, x_fp=x_fp, q_B=q_B, q_C=q_C, dt=dt, z=z, y=y,
                         normed=normed, y_i8=y_i8, out=out, b_fp=keyside_kwargs.get("b_fp"))
        return out

    def _in_project(self, hidden_states):
        """(codes or None, projected)."""
        s = getattr(self.in_proj, "input_scale", None)
        if s is None or not hasattr(self.in_proj, "forward_int8"):
            return None, self.in_proj(hidden_states)
        h_i8 = _fused_fp16_to_int8(_lib.rows16(hidden_states.reshape(-1, hidden_states.shape[-1])), s, clamp_min=-128.0,
                                   reciprocal=False).view(hidden_states.shape)
        return h_i8, self.in_proj.forward_int8(h_i8, s)

    def _split(self, projected):
        """z0, x0 (the MLP's halves, mostly of no width), z, xBC, dt."""
        d_mlp = (projected.shape[-1] - self.d_ssm - self.conv_dim - self.nheads) // 2
        return projected.split([d_mlp, d_mlp, self.d_ssm, self.conv_dim, self.nheads], dim=-1)

    def _finish(self, y, z, z0, x0, host_scale=None):
        """``host_scale``: out_proj's input scale as a number, where reading the tensor would wait for the GPU."""
        out_scale = self.out_proj.input_scale
        quant_scale = out_scale if host_scale is None else host_scale
        d_mlp = z0.shape[-1]
        if d_mlp == 0 and isinstance(self.norm, RMSNormGated):
            y_i8, _ = rmsnorm_gated_qhad(y, z, self.norm.weight, quant_scale, self.norm.eps, self.norm.group_size)
            normed = None
        else:
            normed = self.norm(y, z)
            if d_mlp > 0:
                normed = torch.cat([torch.nn.functional.silu(z0) * x0, normed], dim=-1)
            y_i8, _ = qhad_transform(normed, quant_scale)
        out = self.out_proj.forward_int8(y_i8, out_scale) if hasattr(self.out_proj, "forward_int8") else self.out_proj(y_i8)
        comp_out = getattr(self, "comp_out", None)
        if comp_out is not None:
            out = out + comp_out
        return out, normed, y_i8

    # ---- serving -------------------------------------------------------------------------------------------------------------

    @torch.no_grad()
    def prepare_serving(self):
        """Lays out once what ``prefill`` and ``step`` read beside the projections: the convolution's weights in fp16, A, D and dt_bias in
        fp32 (dequantized as the INT8 kernels do), and out_proj's input scale as a number on the host.  ``allocate_state`` calls it.
        Moving the module, loading a state dict, and exchanging, moving, loading or writing to one of those parameters or the modules that hold
        them undo it."""
        bias = self.conv1d.bias
        self._serving = dict(
            made_of=_AsLaidOut(*self._laid_out()),
            weight=self.conv1d.weight.detach().reshape(self.conv_dim, -1).to(torch.float16, copy=True).contiguous(),
            bias=None if bias is None else bias.detach().to(torch.float16, copy=True),
            A=-torch.exp(self.A_log.float() * self.A_log_scale.float()), D=self.D.float() * self.D_scale.float(),
            dt_bias=None if self.dt_bias is None else self.dt_bias.detach().to(torch.float32, copy=True),
            out_scale=float(self.out_proj.input_scale))

    def _laid_out(self):
        conv = self.conv1d
        return conv.weight, conv.bias, self.A_log, self.A_log_scale, self.D, self.D_scale, self.dt_bias, self.out_proj.input_scale

    def _prepared(self):
        return self._serving is not None and self._serving["made_of"].holds(self._laid_out())

    def _apply(self, fn, *args, **kwargs):
        self._serving = None
        return super()._apply(fn, *args, **kwargs)

    def _load_from_state_dict(self, *args, **kwargs):
        self._serving = None
        return super()._load_from_state_dict(*args, **kwargs)

    def allocate_state(self, num_slots):
        """Zeroed slots for that many sequences, on the module's device."""
        if not self._prepared():
            self.prepare_serving()
        device = self._serving["A"].device
        return Mamba2State(torch.zeros(num_slots, self.d_conv - 1, self.conv_dim, dtype=torch.float16, device=device),
                           torch.zeros(num_slots, self.nheads, self.headdim, self.d_state, dtype=torch.float32, device=device))

    @torch.no_grad()
    def prefill(self, hidden_states, state, slots=None, seq_starts=None, _debug=None):
        """The tokens of prompts, or of the next parts of prompts: ``hidden_states`` fp16 or bf16 (B, L, d_model), or (T, d_model) with
        ``seq_starts`` (n + 1 int32, ascending) for packed prompts of any lengths, or the pair (codes, scale) of its INT8 form.
        ``slots`` (n,) int32: each prompt's place in ``state`` (None: 0 .. n - 1), all different; a negative one marks a prompt that
        starts from zero and leaves nothing.  The state goes on from what the slots hold.  Returns fp16 like hidden_states; rows of
        tokens outside every prompt are undefined."""
        return self._serve(hidden_states, state, slots, seq_starts, False, _debug)

    @torch.no_grad()
    def step(self, hidden_states, state, slots=None, _debug=None):
        """One token of each sequence: ``hidden_states`` (B, d_model), or its (codes, scale) -> (B, d_model).  Entries with a negative
        slot are padding: they touch no state.  Capturable into a graph."""
        return self._serve(hidden_states, state, slots, None, True, _debug)

    def _serve(self, hidden_states, state, slots, seq_starts, single, debug):
        if not self._prepared():
            raise RuntimeError("QuantizedMamba2 is not prepared for serving: call prepare_serving() after the module or a part of it was moved, loaded, "
                               "exchanged or written to")
        w = self._serving
        if isinstance(hidden_states, tuple):
            projected = self.in_proj.forward_int8(*hidden_states)
        else:
            projected = self._in_project(hidden_states.to(torch.float16))[1]
        assert projected.dim() == (2 if single or seq_starts is not None else 3), \
            "hidden_states: (B, L, d_model), (T, d_model) with seq_starts, one token each: (B, d_model)"
        z0, x0, z, xBC, dt = self._split(projected)
        if single:
            xBC = conv1d_step(xBC, state.conv, w["weight"], w["bias"], "silu", slots=slots)
        else:
            xBC = conv1d_prompt(xBC, w["weight"], w["bias"], "silu", state=state.conv, slots=slots, seq_starts=seq_starts)
        gn = self.ngroups * self.d_state
        x, B, C = xBC.split([self.d_ssm, gn, gn], dim=-1)
        # B and C as they are: the rotation and D_qk rescaling of the INT8 path leave C . B unchanged and prepare for codes only
        x = x.unflatten(-1, (self.nheads, self.headdim))
        B, C = (t.unflatten(-1, (self.ngroups, self.d_state)) for t in (B, C))
        kw = dict(dt_bias=w["dt_bias"], dt_softplus=True, dt_limit=self.dt_limit, slots=slots)
        if single:
            y = ssm_step(state.ssm, x, dt, w["A"], B, C, w["D"], **kw)
        else:
            y = ssm_prompt(x, dt, w["A"], B, C, w["D"], state=state.ssm, seq_starts=seq_starts, **kw)
        y = y.flatten(-2)
        out, _, y_i8 = self._finish(y, z, z0, x0, w["out_scale"])
        if debug is not None:
            debug.update(projected=projected, xBC=xBC, dt=dt, z=z, y=y, y_i8=y_i8, out=out)
        return out


class Mamba2Block(nn.Module):
    """A mixer in a residual stream, for serving: r = residual + x and mixer(rmsnorm(r)), the norm's output going to in_proj as the
    INT8 codes that the same pass makes of it.  ``x`` and ``residual`` are what the block in front returned (its mixer's output, not
    yet added, and the stream in fp32); the first block takes the embeddings and None."""

    def __init__(self, mixer: QuantizedMamba2, norm_weight: torch.Tensor, eps=1e-5):
        super().__init__()
        self.mixer, self.eps = mixer, eps
        self.register_buffer("norm_weight", norm_weight.detach().clone())

    def _normed(self, x, residual):
        s = self.mixer.in_proj.input_scale
        codes, scale, r = residual_rmsnorm(x, self.norm_weight, residual, self.eps, quantize="rows" if s is None else s,
                                           residual_dtype=torch.float32 if residual is None else None)
        return (codes, scale), r

    @torch.no_grad()
    def prefill(self, x, residual, state, slots=None, seq_starts=None):
        """-> (the mixer's output, residual); arguments as in ``QuantizedMamba2.prefill``."""
        codes, r = self._normed(x, residual)
        return self.mixer.prefill(codes, state, slots, seq_starts), r

    @torch.no_grad()
    def step(self, x, residual, state, slots=None):
        codes, r = self._normed(x, residual)
        return self.mixer.step(codes, state, slots), r


def random_calibrated_mixer(*, d_model, nheads, headdim, d_state, ngroups, chunk_size, d_conv=4, batch=2, seqlen=512,
                            keyside=False, rotate=True, seed=0, device="cuda", linear=Int8InputLinear):
    """A QuantizedMamba2 with random fp16 weights, calibrated on one synthetic batch (static absmax scales), for tests
    and timing: there are no checkpoints here.  Returns (module, calibration hidden states)."""
    import math
    from types import SimpleNamespace

    from linquant_amd import hadamard_utils as HU
    from linquant_amd.calibration import Mamba2Shape, calibrate_mamba2, mamba2_params

    g = torch.Generator().manual_seed(seed)
    d_ssm, gn = nheads * headdim, ngroups * d_state
    conv_dim = d_ssm + 2 * gn
    d_in = 2 * d_ssm + 2 * gn + nheads
    in_proj = nn.Linear(d_model, d_in, bias=False)
    out_proj = nn.Linear(d_ssm, d_model, bias=False)
    conv1d = nn.Conv1d(conv_dim, conv_dim, d_conv, groups=conv_dim, padding=d_conv - 1)
    with torch.no_grad():
        in_proj.weight.copy_(torch.randn(d_in, d_model, generator=g) / math.sqrt(d_model))
        in_proj.weight[-nheads:] *= 0.5                                  # raw dt rows: N(-2, 0.5) after the shift below
        out_proj.weight.copy_(torch.randn(d_model, d_ssm, generator=g) / math.sqrt(d_ssm))
        conv1d.weight.copy_(torch.randn(conv_dim, 1, d_conv, generator=g) * 0.5)
        conv1d.bias.copy_(torch.randn(conv_dim, generator=g) * 0.1)
    shape = Mamba2Shape(batch=batch, seqlen=seqlen, nheads=nheads, headdim=headdim, dstate=d_state, ngroups=ngroups,
                        chunk=chunk_size)
    params = mamba2_params(shape, seed=seed + 42, device=device)
    params["dt_bias"] = torch.full((nheads,), -2.0, dtype=torch.float32, device=device)
    norm = RMSNormGated(d_ssm, eps=1e-5, group_size=d_ssm // ngroups, device=device)
    with torch.no_grad():
        norm.weight.copy_((1 + 0.1 * torch.randn(d_ssm, generator=g)).to(device))
    hidden = torch.randn(batch, seqlen, d_model, generator=g).to(torch.float16).to(device)

    # calibration pass in plain torch: projection, conv + SiLU, then the SSD observers
    in_scale = hidden.float().abs().amax() / 127.0
    w_in = in_proj.weight.to(device).half()
    proj = torch.nn.functional.linear(hidden, w_in)
    z, xBC_raw, dt_raw = proj.split([d_ssm, conv_dim, nheads], dim=-1)
    xc = torch.nn.functional.conv1d(xBC_raw.float().transpose(1, 2), conv1d.weight.to(device).float(),
                                    conv1d.bias.to(device).float(), padding=d_conv - 1, groups=conv_dim)[..., :seqlen]
    xBC = torch.nn.functional.silu(xc).transpose(1, 2).half().contiguous()
    if not rotate:
        params["r_signs"] = torch.ones_like(params["r_signs"])
    sc = calibrate_mamba2(shape, xBC, dt_raw, params)
    scales = dict(B_scale=sc["B_scale"], B_inv_scale=sc["B_inv_scale"], C_scale=sc["C_scale"], C_inv_scale=sc["C_inv_scale"],
                  A_log_scale=params["A_log_scale"], D_scale=params["D_scale"], A_log_inv_scale=1.0, D_inv_scale=1.0,
                  in_proj_input_scale=in_scale, out_proj_input_scale=torch.tensor(1.0))
    original = SimpleNamespace(nheads=nheads, headdim=headdim, d_model=d_model, d_state=d_state, ngroups=ngroups,
                               d_conv=d_conv, chunk_size=chunk_size, in_proj=in_proj.to(device), out_proj=out_proj.to(device),
                               conv1d=conv1d.to(device).half(), norm=norm, A_log=params["A_log"].float(), D=params["D"].float(),
                               dt_bias=params["dt_bias"], layer_idx=0)
    m = QuantizedMamba2.from_fp16(original, scales, params["r_signs"], linear)
    for name in ("alpha_hp", "bscale_g", "static_state_scale", "static_cb_scale"):
        m.register_buffer(name, sc[name])
    if keyside:
        m.keyside = True
        m.register_buffer("x_quant_scale_hp", sc["x_scale_hp"])
        m.register_buffer("b_gate_scale", sc["b_gate_scale"])
    m = m.to(device)
    # out_proj input scale: absmax of the rotated normalized activations of the calibration batch
    small = HU.small_order(d_ssm)
    if small != 1 and small not in HU._SMALL:
        HU.register_hadamard(small, HU.hadamard_matrix(small))
    dbg = {}
    plain = m.norm
    m.norm = _Unfused(plain)
    m(hidden, _debug=dbg)
    m.norm = plain
    G = torch.from_numpy(HU.chunk_matrix(d_ssm).astype("float32")).to(device)
    rows = dbg["normed"].float().reshape(-1, d_ssm // 128, 128)
    H128 = torch.from_numpy(HU.sylvester(128).astype("float32")).to(device)
    rot = torch.einsum("pc,rci->rpi", G, rows) @ H128
    m.out_proj.input_scale.copy_(rot.abs().amax() / math.sqrt(d_ssm) / 127.0)
    return m, hidden


class _Unfused(nn.Module):
    """Wraps a norm so that the mixer takes the two-launch route (norm, then Hadamard + INT8)."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x, z=None):
        return self.inner(x, z)
