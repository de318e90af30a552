"""Per-row int8 quantiser on the GPU (app/convert_final.py:17-21) and synthetic weights.

``q8_rows`` produces the same int8 codes and bf16 scales as the reference converter
(codes from the unrounded fp32 scale, round half to even, clamp to +-127).
``synthetic_weights`` builds a random-init model in the ``mula_int8.safetensors`` layout
(names of app/convert_final.py:32-47 and app/engine.py:110-114, :249-262), quantised on
the device with that kernel -- there is no network to fetch trained weights.
"""
from __future__ import annotations

import torch

from . import _ffi
from .kernels import INT_MOST, _call_on, stream_ptr

AUDIO_VOCAB = 8197
N_CB = 8


def q8_rows(t: torch.Tensor):
    """t [N, K] (any float dtype, ROCm device) -> (q8 int8 [N, K], s8 bfloat16 [N])."""
    if not t.is_cuda:
        raise RuntimeError("q8_rows runs on a ROCm GPU tensor")
    tf = t.float().contiguous()
    N, K = tf.shape
    q = torch.empty(N, K, device=tf.device, dtype=torch.int8)
    s = torch.empty(N, device=tf.device, dtype=torch.bfloat16)
    _ffi.call("ecd_quantize_rows_i8", tf.data_ptr(), q.data_ptr(), s.data_ptr(), None, N, K,
              stream_ptr(tf.device))
    return q, s


_Q4_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def q4_rows(t: torch.Tensor, group: int = 128, zeros: bool = False):
    """t [N, K] (float32, float16 or bfloat16, ROCm device) -> (q4 uint8 [N, K / 2], s4 float16 [N, K / group rounded up],
    z4 uint8 of the same shape or None): weights of 4 bits with a scale, and with ``zeros`` a zero point, for each ``group``
    (32, 64 or 128) of a row.  Element 2 i is in the low half of byte i and stands for s4 (code - z4), z4 = 8 without
    zeros; include/ecdecode.h gives the rounding.  K is a multiple of 64."""
    if not t.is_cuda:
        raise RuntimeError("q4_rows runs on a ROCm GPU tensor")
    if t.dtype not in _Q4_TYPES:
        raise TypeError(f"q4_rows: expected float32, float16 or bfloat16, got {t.dtype}")
    if t.dim() != 2 or t.shape[1] % 64 or not 0 < t.shape[1] <= INT_MOST or not 0 < t.shape[0] <= INT_MOST:
        raise ValueError("q4_rows: t must be [N, K] with K a multiple of 64")
    if group not in (32, 64, 128):
        raise ValueError("q4_rows: the group must be 32, 64 or 128")
    t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone()
    N, K = t.shape
    q = torch.empty(N, K // 2, device=t.device, dtype=torch.uint8)
    s = torch.empty(N, -(-K // group), device=t.device, dtype=torch.float16)
    z = torch.empty_like(s, dtype=torch.uint8) if zeros else None
    _call_on(t.device, "ecd_quantize_rows_q4", t.data_ptr(), _Q4_TYPES[t.dtype], q.data_ptr(), s.data_ptr(),
             None if z is None else z.data_ptr(), N, K, int(group))
    return q, s, z


def _stack_shapes(prefix, cfg):
    D, H, Hk = cfg["dim"], cfg["heads"], cfg["kv_heads"]
    hd = D // H
    F = cfg.get("ffn", 8192)
    for i in range(cfg["layers"]):
        pre = f"{prefix}.layers.{i}."
        yield pre + "attn.q_proj.weight", (H * hd, D)
        yield pre + "attn.k_proj.weight", (Hk * hd, D)
        yield pre + "attn.v_proj.weight", (Hk * hd, D)
        yield pre + "attn.output_proj.weight", (D, H * hd)
        yield pre + "mlp.w1.weight", (F, D)
        yield pre + "mlp.w3.weight", (F, D)
        yield pre + "mlp.w2.weight", (D, F)


def _stack_norms(prefix, cfg):
    for i in range(cfg["layers"]):
        yield f"{prefix}.layers.{i}.sa_norm.scale", cfg["dim"]
        yield f"{prefix}.layers.{i}.mlp_norm.scale", cfg["dim"]
    yield f"{prefix}.norm.scale", cfg["dim"]


def weight_shapes(backbone: dict, decoder: dict, text_vocab: int = 1024):
    """(quantised tensors {name: (N, K)}, bf16 tensors {name: shape}) of the file layout."""
    Db, Dd = backbone["dim"], decoder["dim"]
    lin = dict(_stack_shapes("backbone", backbone))
    lin.update(_stack_shapes("decoder", decoder))
    lin["projection.weight"] = (Dd, Db)
    lin["codebook0_head.weight"] = (AUDIO_VOCAB, Db)
    for i in range(N_CB - 1):
        lin[f"audio_head.{i}"] = (AUDIO_VOCAB, Dd)
    lin["audio_embeddings.weight"] = (N_CB * AUDIO_VOCAB, Db)
    lin["text_embeddings.weight"] = (text_vocab, Db)
    dense = {n: (d,) for n, d in _stack_norms("backbone", backbone)}
    dense.update({n: (d,) for n, d in _stack_norms("decoder", decoder)})
    dense["unconditional_text_embedding.weight"] = (1, Db)
    dense["muq_linear.bias"] = (Db,)
    return lin, dense


def to_q4(weights: dict, group: int = 128, zeros: bool = False, device="cuda", stack: str = "backbone") -> dict:
    """A model's int8 weights with the linear layers of ``stack`` in 4 bits (their values requantised group by group): the
    names ``<name>.q8`` / ``.s8`` become ``<name>.q4`` / ``.s4`` (/ ``.z4``)."""
    out = {}
    for k, v in weights.items():
        name, kind = k.rsplit(".", 1)
        if not name.startswith(f"{stack}.layers.") or kind not in ("q8", "s8"):
            out[k] = v
        elif kind == "q8":
            w = v.to(device).float() * weights[name + ".s8"].to(device).float()[:, None]
            q, s, z = q4_rows(w, group, zeros)
            out[name + ".q4"], out[name + ".s4"] = q, s
            if zeros:
                out[name + ".z4"] = z
    return out


@torch.no_grad()
def synthetic_weights(backbone: dict, decoder: dict, device="cuda", seed: int = 0,
                      std: float = 0.02, emb_std: float = 1.0, text_vocab: int = 1024):
    """Random-init weights in the int8 file layout: linear weights ~ N(0, std), embedding
    tables ~ N(0, emb_std), norm scales 1 + N(0, 0.02), quantised per row on the GPU."""
    dev = torch.device(device)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    lin, dense = weight_shapes(backbone, decoder, text_vocab)
    out = {}
    for name, (N, K) in lin.items():
        sd = emb_std if "embeddings" in name else std
        w = torch.randn(N, K, generator=g, device=dev) * sd
        out[name + ".q8"], out[name + ".s8"] = q8_rows(w)
        del w
    for name, shp in dense.items():
        if name.endswith(".scale"):
            t = 1.0 + 0.02 * torch.randn(*shp, generator=g, device=dev)
        else:
            t = torch.randn(*shp, generator=g, device=dev) * (emb_std if "embedding" in name else std)
        out[name] = t.to(torch.bfloat16)
    return out
