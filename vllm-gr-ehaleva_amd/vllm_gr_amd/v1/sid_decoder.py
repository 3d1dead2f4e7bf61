"""Random-init Qwen-style decoder for end-to-end semantic-ID beam decode.

The reference serves a Qwen3 checkpoint through vLLM's model executor
(vllm==0.14, not vendored; the semantic-ID tasks use Qwen3 chat templates,
benchmarks/open_one_rec/tasks/recommendation/config.py:19).  This is the
same architecture, sized by a :class:`DecoderConfig`, with weights drawn
from N(0, std) -- there are no checkpoints here:

* token embedding, tied to the lm_head by default;
* per layer: RMSNorm, q/k/v projections (no bias), per-head RMSNorm of q and
  k, rotary embedding with rotate-half pairing (theta 1e6) at the positions
  the caller gives, attention through the BeamAttention backend, o
  projection, residual add; RMSNorm, SwiGLU MLP (silu(gate) * up, down) or,
  with ``num_experts``, a router and the SwiGLU layers of the experts it
  chooses for each token, residual add;
* final RMSNorm; logits = lm_head products in ``cfg.dtype``, widened to float32.

The projections of a decode step's qkv, o, gate_up (with its SiLU gate) and
lm_head are gr_linear where that is the faster (up to 512 rows, from at most 2048
features: ``_own_sizes``); the others are ``torch.nn.functional.linear`` (hipBLASLt on ROCm).  The
elementwise stages are fused HIP kernels (include/gr_decoder.h): residual add
+ RMSNorm, per-head q/k RMSNorm + rotary + K/V cache write through the slot
mapping, and the SiLU-gated product.  With weights from
``quantize_weights`` a layer's projections and experts are e4m3 in blocks of 128 x 128
(include/gr_experts.h), their inputs quantised token by token.  Attention is
:class:`BeamAttentionImpl.forward`, the call vLLM's Attention layer makes
(beam_attn.py:703-755), with the K/V already written (key/value None).
Positions follow the reference's rule (a beam's j-th suffix token sits at prefix_len + j,
engine_core_patch.py:362-365); logits are taken for one row per beam, the
beam's newest token (:367-369).
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from .. import ops
from .attention.backends.beam_attn import BeamAttentionImpl


@dataclass(frozen=True)
class DecoderConfig:
    num_layers: int = 28
    hidden: int = 2048
    num_heads: int = 16
    num_kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 6144
    vocab: int = 8192
    rope_theta: float = 1.0e6
    rms_eps: float = 1.0e-6
    tie_embeddings: bool = True
    init_std: float = 0.02
    dtype: torch.dtype = torch.bfloat16
    # experts in place of the MLP (0: none; 16-bit dtypes): each token's
    # experts_per_token of them, chosen by route_experts with these options
    num_experts: int = 0
    experts_per_token: int = 8
    expert_ffn: int = 768
    router_score: str = "softmax"
    router_bias: bool = False
    router_groups: int = 1
    router_top_groups: int = 1
    router_renormalize: bool = True
    router_scale: float = 1.0

    @property
    def q_size(self) -> int:
        return self.num_heads * self.head_dim

    @property
    def kv_size(self) -> int:
        return self.num_kv_heads * self.head_dim

    def num_params(self) -> int:
        H, L = self.hidden, self.num_layers
        mlp = 3 * H * self.ffn
        if self.num_experts:
            mlp = self.num_experts * (3 * H * self.expert_ffn + H + (1 if self.router_bias else 0))
        per_layer = H * (self.q_size + 2 * self.kv_size) + self.q_size * H + mlp + 2 * H + 2 * self.head_dim
        emb = self.vocab * H * (1 if self.tie_embeddings else 2)
        return L * per_layer + emb + H


#: the 28-layer, 2048-hidden, 16/8-head, 6144-FFN, 8192-token decoder
SID_DECODER_1P7B = DecoderConfig()


def init_weights(cfg: DecoderConfig, seed: int, device="cpu") -> dict[str, torch.Tensor]:
    """Weights in nn.Linear layout ``[out, in]``, drawn from one generator on
    ``device`` in a fixed order (embedding, then per layer qkv, o, gate_up,
    down; with experts router, expert_gate_up ``[E, 2 F, H]``, expert_down ``[E, H,
    F]``), N(0, init_std) in float32 rounded to ``cfg.dtype``; norm weights
    are ones, a router's bias zeros (float32).  The same seed and device give the
    same weights."""
    dev = torch.device(device)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape):
        w = torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)
        return w.mul_(cfg.init_std).to(cfg.dtype)

    ones = lambda n: torch.ones(n, device=dev, dtype=cfg.dtype)
    H = cfg.hidden
    w = {"embed": normal(cfg.vocab, H)}
    for i in range(cfg.num_layers):
        p = f"layers.{i}."
        w[p + "qkv"] = normal(cfg.q_size + 2 * cfg.kv_size, H)
        w[p + "o"] = normal(H, cfg.q_size)
        if cfg.num_experts:
            E, F_ = cfg.num_experts, cfg.expert_ffn
            w[p + "router"] = normal(E, H)
            if cfg.router_bias:
                w[p + "router_bias"] = torch.zeros(E, device=dev)
            w[p + "expert_gate_up"] = normal(E, 2 * F_, H)
            w[p + "expert_down"] = normal(E, H, F_)
        else:
            w[p + "gate_up"] = normal(2 * cfg.ffn, H)
            w[p + "down"] = normal(H, cfg.ffn)
        w[p + "input_norm"] = ones(H)
        w[p + "post_norm"] = ones(H)
        w[p + "q_norm"] = ones(cfg.head_dim)
        w[p + "k_norm"] = ones(cfg.head_dim)
    w["final_norm"] = ones(H)
    w["lm_head"] = w["embed"] if cfg.tie_embeddings else normal(cfg.vocab, H)
    return w


def quantize_blocks(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``w [..., N, K]`` as e4m3 with a float32 scale for each block of 128 x 128
    (``[..., ceil(N / 128), ceil(K / 128)]``): the block's largest magnitude over
    448, at least 2^-80, as gr_quant_fp8 scales a row's groups."""
    N, K = w.shape[-2:]
    nb, kb = -(-N // ops.FP8_BLOCK), -(-K // ops.FP8_BLOCK)
    x = F.pad(w.float(), (0, kb * ops.FP8_BLOCK - K, 0, nb * ops.FP8_BLOCK - N))
    x = x.unflatten(-1, (kb, ops.FP8_BLOCK)).unflatten(-3, (nb, ops.FP8_BLOCK))
    scale = (x.abs().amax((-3, -1)) / 448.0).clamp_min(2.0 ** -80)
    x = (x / scale[..., :, None, :, None]).flatten(-2).flatten(-3, -2)[..., :N, :K]
    return x.to(torch.float8_e4m3fn).contiguous(), scale.contiguous()


_QUANTIZED = ("qkv", "o", "gate_up", "down", "expert_gate_up", "expert_down")


def quantize_weights(weights: dict[str, torch.Tensor]) -> dict[str, torch.Tensor]:
    """A decoder's weights with every layer's projections and experts in e4m3 and
    their scales beside them (``<name>_scale``); gate and up are scaled apart.
    Embedding, lm_head, norms and router stay as they are, and so does what has its
    scales already."""
    out = {}
    for name, w in weights.items():
        kind = name.rsplit(".", 1)[-1]
        if not name.startswith("layers.") or kind not in _QUANTIZED or name + "_scale" in weights:
            out[name] = w
        elif kind.endswith("gate_up"):
            w8, scale = quantize_blocks(w.unflatten(-2, (2, w.shape[-2] // 2)))
            out[name], out[name + "_scale"] = w8.flatten(-3, -2), scale.flatten(-3, -2).contiguous()
        else:
            out[name], out[name + "_scale"] = quantize_blocks(w)
    return out


class RotaryEmbedding:
    """Tables of the rotate-half rotary embedding: pair (i, i + D/2) turns by
    ``pos * theta^(-2i/D)``; cos/sin ``[max_pos, D/2]`` evaluated in float64
    and stored as float32 on the device (read by gr_qk_norm_rope_cache)."""

    def __init__(self, head_dim: int, theta: float, max_pos: int, device):
        half = head_dim // 2
        inv = 1.0 / (theta ** (torch.arange(0, half, dtype=torch.float64) * 2.0 / head_dim))
        ang = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv[None]
        self.cos = ang.cos().float().to(device)
        self.sin = ang.sin().float().to(device)
        self.max_pos = max_pos


def _plain(*ts: torch.Tensor) -> bool:
    """Whether a kernel on the tensors' addresses can stand in for a torch
    operation: ordinary tensors, and nothing that follows torch operations --
    an autograd graph, forward mode, vmap and the other function transforms, a
    dispatch mode (fake tensors, tracing) or a compiler -- would miss it.  (The
    layers of ``forward`` run such kernels throughout; ``compute_logits`` is one
    product and keeps what the torch product does.)"""
    return (all(type(t) in (torch.Tensor, torch.nn.Parameter) for t in ts)
            and not (torch.is_grad_enabled() and any(t.requires_grad for t in ts))
            and torch.autograd.forward_ad._current_level < 0 and torch._C._functorch.peek_interpreter_stack() is None
            and torch._C._len_torch_dispatch_stack() == 0
            and not torch.jit.is_tracing() and not torch.compiler.is_compiling())


def _own_sizes(m: int, rows: int, k: int, swiglu: bool) -> bool:
    """Whether gr_linear takes a projection of ``m`` rows by ``rows`` weight rows
    of ``k`` features.

    Measured with cold weights over 1 to 512 rows, 512 to 151936 weight rows and
    512 to 2048 features, own time / the library's (SwiGLU: its product and the
    gate kernel's):

    * workgroups that fill the chip once (128 x 192 tiles, column tiles whole on
      one of the 8 XCDs of 32 CUs) and SwiGLU, 0.37 to 0.91, or at most 1024
      features, 0.44 to 1.00 (of random sizes 1 in 100 up to 1.17).  In more rounds
      0.75 to 1.60, SwiGLU 0.43 to 1.35;
    * one round and more features: 0.51 to 1.00, but not where few columns leave
      most CUs idle and the rows fill the library's tiles (33 to 128 rows: 512
      columns 0.97 to 1.04, 1024 0.85 to 1.09, 2048 at 64 and 128 rows 0.99 to
      1.03), and not around its best fits past 1536 features (337 to 384 rows, 3072
      and 4096 columns 1.01 to 1.08; 257 to 315 rows, 5664 to 6512 columns 1.04 to
      1.10, though 0.80 to 0.89 at 320 to 340);
    * up to 100 rows the weights' way from memory is the time, also in more
      rounds: 0.55 to 0.98 past 1024 features;
    * above the limits: 768 rows, SwiGLU 2048 in, 6144 out 53 us against 44; 6144
      in, 2048 out, 8 rows 21 against 12."""
    if m > 512 or k > 2048:
        return False
    one_round = -(-m // 128) * -(-rows // (8 * 192)) <= 32
    if swiglu or k <= 1024:
        return one_round
    if not one_round:
        return m <= 100
    if m <= 32:
        return True
    if m <= 128:
        return rows > 2048 or (rows > 1024 and m % 64 != 0)
    if k > 1536 and 256 < m <= 384 and 2560 < rows < 8192:
        return rows <= 5120 and m <= 336
    return rows > 512


def _own_linear(x: torch.Tensor, w: torch.Tensor, swiglu: bool = False) -> bool:
    return _own_sizes(x.shape[0], *w.shape, swiglu) and ops.linear_supported(x, w, swiglu)


def _linear(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    return ops.linear(x, w) if _own_linear(x, w) else F.linear(x, w)


def _swiglu(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    return ops.linear(x, w, swiglu=True) if _own_linear(x, w, True) else ops.silu_mul(F.linear(x, w))


def _check_experts(cfg: DecoderConfig) -> None:
    """Refuses what route_experts and expert_mlp would refuse in the first forward."""
    E, k, groups, top = cfg.num_experts, cfg.experts_per_token, cfg.router_groups, cfg.router_top_groups
    if cfg.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("experts need a 16-bit dtype")
    if cfg.hidden % 16 or cfg.expert_ffn % 16 or cfg.expert_ffn < 1 or E > 1024:
        raise ValueError("experts need hidden and expert_ffn in multiples of 16, and are at most 1024")
    if cfg.router_score not in ("softmax", "sigmoid"):
        raise ValueError("router_score must be 'softmax' or 'sigmoid'")
    if not 1 <= top <= groups <= 64 or E % groups or not 1 <= k <= min(64, E // groups * top):
        raise ValueError("experts_per_token (64 at most) are chosen from router_top_groups of router_groups equal groups")


def _check_quantized(cfg: DecoderConfig, weights: dict[str, torch.Tensor]) -> None:
    """Refuses 8-bit weights that the products would refuse in the first forward."""
    names = ("expert_gate_up", "expert_down") if cfg.num_experts else ("gate_up", "down")
    for i in range(cfg.num_layers):
        p = f"layers.{i}."
        for name in (p + "qkv", p + "o", p + names[0], p + names[1]):
            w, scale = weights.get(name), weights.get(name + "_scale")
            if w is None or (scale is None and w.dtype != torch.float8_e4m3fn):
                continue
            if scale is None or w.dtype != torch.float8_e4m3fn:
                raise ValueError(f"{name}: float8_e4m3fn weights and {name}_scale go together")
            parts = 2 if name.endswith("gate_up") else 1  # gate's rows, then up's
            N, K = w.shape[-2] // parts, w.shape[-1]
            if K % 16 or w.shape[-2] % parts or (parts == 2 and N % 16):
                raise ValueError(f"{name}: 8-bit weights need sizes in multiples of 16, not {list(w.shape)}")
            blocks = [-(-n // ops.FP8_BLOCK) for n in (N, K)]
            shape = (*w.shape[:-2], parts * blocks[0], blocks[1])
            if scale.shape != shape or scale.dtype != torch.float32 or not scale.is_contiguous():
                raise ValueError(f"{name}_scale must be a contiguous float32 {list(shape)} tensor")
        if (p + names[0] + "_scale" in weights) != (p + names[1] + "_scale" in weights):
            raise ValueError(f"{p}{names[0]} and {p}{names[1]} are 8-bit together or not at all")


class SidDecoder:
    """The decoder's forward over a flat batch of tokens.

    ``forward(input_ids, positions, attn_metadata, kv_caches)`` runs every
    layer; ``kv_caches[i]`` is layer i's ``[2, num_blocks, block_size, Hkv,
    D]`` cache and ``attn_metadata`` the backend metadata of the batch (its
    slot mapping says where each token's K/V is written).  Positions lie
    below ``max_position`` (the rotary table's length; the kernel flags and
    skips a token beyond it).  Returns the final normalised hidden states
    ``[T, hidden]``; :meth:`compute_logits` maps selected rows to float32
    logits."""

    def __init__(self, cfg: DecoderConfig, weights: dict[str, torch.Tensor], *, max_position: int = 32768):
        if cfg.num_experts:
            _check_experts(cfg)
        _check_quantized(cfg, weights)
        self.cfg = cfg
        self.w = weights
        dev = weights["embed"].device
        self.rope = RotaryEmbedding(cfg.head_dim, cfg.rope_theta, max_position, dev)
        self.layer_names = [f"model.layers.{i}.self_attn.attn" for i in range(cfg.num_layers)]
        self.attn = [BeamAttentionImpl(cfg.num_heads, cfg.head_dim, 1.0 / math.sqrt(cfg.head_dim),
                                       cfg.num_kv_heads, None, None, "auto")
                     for _ in range(cfg.num_layers)]

    @property
    def device(self) -> torch.device:
        return self.w["embed"].device

    def _project(self, x: torch.Tensor, name: str) -> torch.Tensor:
        w, scale = self.w[name], self.w.get(name + "_scale")
        if scale is None:
            return _linear(x, w)
        return ops.linear_fp8(*ops.quant_fp8(x), w, scale, out_dtype=x.dtype)

    def _mlp(self, x: torch.Tensor, p: str) -> torch.Tensor:
        w, cfg = self.w, self.cfg
        if cfg.num_experts:
            router = w[p + "router"]
            # the scores' order decides: float32 logits
            logits = (ops.linear(x, router, out_f32=True) if _own_linear(x, router)
                      else F.linear(x.float(), router.float()))
            weights, ids = ops.route_experts(
                logits, cfg.experts_per_token, score=cfg.router_score, bias=w.get(p + "router_bias"),
                num_groups=cfg.router_groups, top_groups=cfg.router_top_groups,
                renormalize=cfg.router_renormalize, scale=cfg.router_scale)
            return ops.expert_mlp(x, w[p + "expert_gate_up"], w[p + "expert_down"], weights, ids,
                                  gate_up_scale=w.get(p + "expert_gate_up_scale"),
                                  down_scale=w.get(p + "expert_down_scale"))
        scale = w.get(p + "gate_up_scale")
        if scale is None:
            return _linear(_swiglu(x, w[p + "gate_up"]), w[p + "down"])
        act = ops.linear_fp8(*ops.quant_fp8(x), w[p + "gate_up"], scale, swiglu=True, quantized=True)
        return ops.linear_fp8(*act, w[p + "down"], w[p + "down_scale"], out_dtype=x.dtype)

    def forward(self, input_ids: torch.Tensor, positions: torch.Tensor, attn_metadata,
                kv_caches) -> torch.Tensor:
        cfg, w, eps = self.cfg, self.w, self.cfg.rms_eps
        T = input_ids.shape[0]
        slots = attn_metadata.slot_mapping if attn_metadata is not None else None
        status = attn_metadata.status if attn_metadata is not None else None
        h = w["embed"][input_ids]  # the residual stream
        x = ops.rms_norm(h, w["layers.0.input_norm"], eps)
        mlp = None
        for i in range(cfg.num_layers):
            p = f"layers.{i}."
            if i:
                x = ops.rms_norm(mlp, w[p + "input_norm"], eps, residual=h, out=x)
            qkv = self._project(x, p + "qkv")
            k_cache, v_cache = ops.split_kv_cache(kv_caches[i])
            q = ops.qk_norm_rope_cache(qkv, positions, self.rope.cos, self.rope.sin, w[p + "q_norm"],
                                       w[p + "k_norm"], k_cache, v_cache, slots, num_q_heads=cfg.num_heads,
                                       num_kv_heads=cfg.num_kv_heads, head_dim=cfg.head_dim, eps=eps,
                                       status=status)
            attn = torch.empty_like(q)
            self.attn[i].forward(None, q, None, None, kv_caches[i], attn_metadata, output=attn)
            x = ops.rms_norm(self._project(attn.view(T, cfg.q_size), p + "o"), w[p + "post_norm"], eps,
                             residual=h, out=x)
            mlp = self._mlp(x, p)
        return ops.rms_norm(mlp, w["final_norm"], eps, residual=h)

    def compute_logits(self, hidden: torch.Tensor) -> torch.Tensor:
        # the model type's values on either path: scores and their ties do not
        # depend on how many rows share the step
        w = self.w["lm_head"]
        if _plain(hidden, w) and _own_linear(hidden, w):
            return ops.linear(hidden, w, out_f32=True, rounded=True)
        return F.linear(hidden, w).float()
