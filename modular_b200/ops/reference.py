"""Plain PyTorch implementations of every op in :mod:`modular_b200.ops`.

They define the semantics the CUDA kernels are tested against (fp32 math, the same
rounding points) and are the execution path on CPU-only machines.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def linear(x, w, residual=None, out_dtype=None):
    y = (x.float() @ w.float().t()).to(out_dtype or x.dtype)
    if residual is not None:
        y = (y.float() + residual.float()).to(y.dtype)
    return y


def linear_swiglu(x, w_gate_up):
    inter = w_gate_up.shape[0] // 2
    g = x.float() @ w_gate_up[:inter].float().t()
    u = x.float() @ w_gate_up[inter:].float().t()
    return (F.silu(g) * u).to(x.dtype)


def rms_norm(x, w, eps, weight_offset=0.0, multiply_before_cast=False):
    xf = x.float()
    n = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    wf = w.float() + weight_offset
    if multiply_before_cast:
        return (n * wf).to(x.dtype)
    return (n.to(x.dtype).float() * wf).to(x.dtype)


def add_rms_norm(x, residual, w, eps, weight_offset=0.0, multiply_before_cast=False):
    h = (x.float() + residual.float()).to(x.dtype)
    return rms_norm(h, w, eps, weight_offset, multiply_before_cast), h


def silu_mul(gate_up):
    inter = gate_up.shape[-1] // 2
    g, u = gate_up[..., :inter].float(), gate_up[..., inter:].float()
    return (F.silu(g) * u).to(gate_up.dtype)


def xielu(x, up: float, down: float):
    z = x.float()
    low = z.clamp(max=0.0)
    return torch.where(z > 0, up * z * z, down * (torch.expm1(low) - low)).add(0.5 * z).to(x.dtype)


def gelu_tanh(x):
    return F.gelu(x.float(), approximate="tanh").to(x.dtype)


def embedding(ids, table, vocab_start=0):
    local = ids - vocab_start
    ok = (local >= 0) & (local < table.shape[0])
    out = table[local.clamp(0, table.shape[0] - 1)]
    return out * ok.unsqueeze(-1).to(out.dtype)


def apply_rope(x, cos, sin, interleaved=False):
    """x: [T, H, D]; cos/sin: [T, D/2]."""
    xf = x.float()
    c, s = cos.unsqueeze(1).float(), sin.unsqueeze(1).float()
    if interleaved:
        a, b = xf[..., 0::2], xf[..., 1::2]
        out = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    else:
        half = x.shape[-1] // 2
        a, b = xf[..., :half], xf[..., half:]
        out = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    return out.to(x.dtype)


def rope_kv_store(qkv, positions, slots, cos_sin, k_cache, v_cache, n_q, n_kv, head_dim,
                  interleaved=False):
    """In place: rotates Q (and K) inside ``qkv`` and scatters K/V into the paged cache.

    k_cache / v_cache: [pages, n_kv, page_size, head_dim] views of one layer.
    """
    T = qkv.shape[0]
    half = head_dim // 2
    cs = cos_sin[positions.long()]
    cos, sin = cs[:, :half], cs[:, half:]
    q = qkv[:, : n_q * head_dim].view(T, n_q, head_dim)
    k = qkv[:, n_q * head_dim : (n_q + n_kv) * head_dim].view(T, n_kv, head_dim)
    v = qkv[:, (n_q + n_kv) * head_dim :].view(T, n_kv, head_dim)
    q.copy_(apply_rope(q, cos, sin, interleaved))
    k_rot = apply_rope(k, cos, sin, interleaved)
    page_size = k_cache.shape[2]
    ok = slots >= 0
    pg = torch.div(slots.clamp(min=0), page_size, rounding_mode="floor")
    off = slots.clamp(min=0) % page_size
    k_cache[pg[ok], :, off[ok]] = k_rot[ok].to(k_cache.dtype)
    v_cache[pg[ok], :, off[ok]] = v[ok].to(v_cache.dtype)


def paged_attention(q, k_cache, v_cache, block_table, q_start, q_len, kv_len, n_q, n_kv,
                    head_dim, scale):
    """Ragged causal attention over a paged cache. q: [T, >= n_q*head_dim] (row stride free)."""
    T = q.shape[0]
    out = torch.zeros(T, n_q * head_dim, dtype=q.dtype, device=q.device)
    G = n_q // n_kv
    page_size = k_cache.shape[2]
    for b in range(block_table.shape[0]):
        qs, ql, kl = int(q_start[b]), int(q_len[b]), int(kv_len[b])
        if ql == 0:
            continue
        n_pages = (kl + page_size - 1) // page_size
        pages = block_table[b, :n_pages].long()
        k = k_cache[pages].permute(1, 0, 2, 3).reshape(n_kv, -1, head_dim)[:, :kl].float()
        v = v_cache[pages].permute(1, 0, 2, 3).reshape(n_kv, -1, head_dim)[:, :kl].float()
        qq = q[qs : qs + ql, : n_q * head_dim].view(ql, n_q, head_dim).float()
        k = k.repeat_interleave(G, dim=0)
        v = v.repeat_interleave(G, dim=0)
        s = torch.einsum("qhd,hkd->hqk", qq, k) * scale
        qi = torch.arange(ql, device=q.device).unsqueeze(1) + (kl - ql)
        ki = torch.arange(kl, device=q.device).unsqueeze(0)
        s = s.masked_fill(ki > qi, float("-inf"))
        p = torch.softmax(s, dim=-1)
        o = torch.einsum("hqk,hkd->qhd", p, v)
        out[qs : qs + ql] = o.reshape(ql, -1).to(q.dtype)
    return out


def argmax(logits):
    return logits.argmax(dim=-1)


def apply_penalties(logits, tok, cnt, offsets, freq=None, pres=None, rep=None):
    for r in range(logits.shape[0]):
        b, e = int(offsets[r]), int(offsets[r + 1])
        if e <= b:
            continue
        t = tok[b:e].long()
        c = cnt[b:e].float()
        x = logits[r, t]
        if rep is not None and float(rep[r]) != 1.0:
            x = torch.where(x > 0, x / rep[r], x * rep[r])
        f = freq[r] if freq is not None else 0.0
        p = pres[r] if pres is not None else 0.0
        x = x - (c > 0).float() * (f * c + p)
        logits[r, t] = x
    return logits


def filtered_probs(logits, temperature, top_k, top_p, min_p):
    """Probability vector the device sampler draws from (used by distribution tests)."""
    x = logits.float() / temperature
    mx = x.max()
    keep = torch.ones_like(x, dtype=torch.bool)
    if top_k and 0 < top_k < x.numel():
        kth = torch.topk(x, top_k).values[-1]
        keep &= x >= kth
    if min_p and min_p > 0:
        keep &= x >= mx + math.log(min_p)
    w = torch.where(keep, torch.exp(x - mx), torch.zeros_like(x))
    if top_p is not None and top_p < 1.0:
        order = torch.argsort(x, descending=True)
        ws = w[order]
        csum = torch.cumsum(ws, 0)
        target = top_p * ws.sum()
        # smallest prefix whose mass reaches the target (ties at the cut stay in)
        n_keep = int((csum < target).sum().item()) + 1
        thr = x[order[min(n_keep, x.numel()) - 1]]
        keep &= x >= thr
        w = torch.where(keep, w, torch.zeros_like(w))
    return w / w.sum()


def sample(logits, temperature=None, top_k=None, top_p=None, min_p=None, generator=None):
    out = torch.empty(logits.shape[0], dtype=torch.long, device=logits.device)
    for r in range(logits.shape[0]):
        T = float(temperature[r]) if temperature is not None else 1.0
        k = int(top_k[r]) if top_k is not None else 0
        if T <= 0 or k == 1:
            out[r] = logits[r].argmax()
            continue
        p = filtered_probs(logits[r], T, k, float(top_p[r]) if top_p is not None else 1.0,
                           float(min_p[r]) if min_p is not None else 0.0)
        out[r] = torch.multinomial(p, 1, generator=generator)[0]
    return out


# ------------------------------------------------------------------ block-scaled fp8
FP8_MAX = 448.0


def quant_fp8_group128(x):
    """Per-token-group (1 x 128) dynamic quantisation. Returns (q float8_e4m3fn [M, K],
    scales fp32 [ceil(K/128), M])."""
    M, K = x.shape
    G = (K + 127) // 128
    xf = torch.zeros(M, G * 128, dtype=torch.float32, device=x.device)
    xf[:, :K] = x.float()
    xg = xf.view(M, G, 128)
    scale = xg.abs().amax(-1).clamp_min(1e-12) / FP8_MAX
    q = (xg / scale.unsqueeze(-1)).clamp(-FP8_MAX, FP8_MAX).view(M, G * 128)[:, :K]
    return q.to(torch.float8_e4m3fn), scale.t().contiguous()


def quant_fp8_weight_block128(w):
    """128x128 block quantisation of a weight [N, K]. Returns (q float8_e4m3fn, scales
    [ceil(N/128), ceil(K/128)]) with scale = amax / 448 (the checkpoint's ``weight_scale_inv``)."""
    N, K = w.shape
    nb, kb = (N + 127) // 128, (K + 127) // 128
    wf = torch.zeros(nb * 128, kb * 128, dtype=torch.float32, device=w.device)
    wf[:N, :K] = w.float()
    blocks = wf.view(nb, 128, kb, 128)
    scale = blocks.abs().amax(dim=(1, 3)).clamp_min(1e-12) / FP8_MAX
    q = (blocks / scale[:, None, :, None]).clamp(-FP8_MAX, FP8_MAX).view(nb * 128, kb * 128)[:N, :K]
    return q.to(torch.float8_e4m3fn).contiguous(), scale.contiguous()


def dequant_fp8_weight_block128(q, scale):
    N, K = q.shape
    s = scale.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return q.float() * s


# ---------------------------------------------------------------------------- nvfp4 (e2m1 values, e4m3 block scales)
_E2M1_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quant_nvfp4_weight(w):
    """NVFP4 quantisation of a weight [N, K] (K % 16 == 0): 4-bit e2m1 values, one e4m3 scale per 16 values along K
    and one fp32 scale per tensor. Returns (packed uint8 [N, K / 2] with the even index in the low nibble, block
    scales float8_e4m3fn [N, K / 16], global scale fp32 scalar tensor); ``w ~ e2m1 * block_scale * global_scale``.
    Reference format: the reference's nvfp4 weights (max/python/max/nn/quant_config.py, kernels
    linalg/matmul/gpu/sm100/block_scaled_matmul.mojo)."""
    N, K = w.shape
    assert K % 16 == 0
    wf = w.float()
    amax = wf.abs().amax().clamp_min(1e-12)
    g = amax / (6.0 * FP8_MAX)                                  # block scales then fit e4m3
    blocks = wf.view(N, K // 16, 16)
    bs = (blocks.abs().amax(-1) / 6.0 / g).clamp(max=FP8_MAX).to(torch.float8_e4m3fn)
    denom = (bs.float() * g).clamp_min(1e-30).unsqueeze(-1)
    x = (blocks / denom).clamp(-6.0, 6.0)
    grid = torch.tensor(_E2M1_VALUES, dtype=torch.float32, device=w.device)
    idx = (x.abs().unsqueeze(-1) - grid).abs().argmin(-1)       # nearest representable magnitude
    code = (idx | ((x < 0).long() << 3)).view(N, K).to(torch.uint8)
    packed = (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()
    return packed, bs.contiguous(), g.reshape(()).clone()


def dequant_nvfp4_weight(packed, block_scale, global_scale):
    N, K2 = packed.shape
    grid = torch.tensor(_E2M1_VALUES, dtype=torch.float32, device=packed.device)
    lo, hi = (packed & 0xF).long(), (packed >> 4).long()
    code = torch.stack((lo, hi), dim=-1).view(N, K2 * 2)
    val = grid[code & 7] * torch.where((code & 8) != 0, -1.0, 1.0)
    s = block_scale.float().repeat_interleave(16, 1) * global_scale.float()
    return val * s


def quant_mxfp8_weight(w):
    """MXFP8 quantisation of a weight [N, K] (K % 32 == 0): e4m3 values with one power-of-two scale per 32 values
    along K. Returns (q float8_e4m3fn [N, K], scales uint8 [N, K / 32] in ue8m0: scale = 2^(byte - 127))."""
    N, K = w.shape
    assert K % 32 == 0
    blocks = w.float().view(N, K // 32, 32)
    amax = blocks.abs().amax(-1).clamp_min(2.0 ** -120)
    e = torch.ceil(torch.log2(amax / FP8_MAX)).clamp(-127, 127)
    q = (blocks / torch.exp2(e).unsqueeze(-1)).clamp(-FP8_MAX, FP8_MAX).view(N, K).to(torch.float8_e4m3fn)
    return q.contiguous(), (e + 127).to(torch.uint8).contiguous()


def dequant_mxfp8_weight(q, scale_bytes):
    s = torch.exp2(scale_bytes.float() - 127.0).repeat_interleave(32, 1)
    return q.float() * s


def linear_fp8_blockscaled(xq, xs, wq, ws, residual=None, out_dtype=torch.bfloat16):
    """fp32 emulation of the block-scaled GEMM: partial sums per 128-wide K group, scaled, added."""
    M, K = xq.shape
    N = wq.shape[0]
    G = (K + 127) // 128
    xf, wf = xq.float(), wq.float()
    y = torch.zeros(M, N, dtype=torch.float32, device=xq.device)
    wsn = ws.repeat_interleave(128, 0)[:N]                      # [N, G]
    for g in range(G):
        k0, k1 = g * 128, min(K, (g + 1) * 128)
        part = xf[:, k0:k1] @ wf[:, k0:k1].t()
        y += part * xs[g].unsqueeze(1) * wsn[:, g].unsqueeze(0)
    y = y.to(out_dtype)
    if residual is not None:
        y = (y.float() + residual.float()).to(out_dtype)
    return y


# ---------------------------------------------------------------------- 8-bit paged key/value cache
FP8_ROW_LEAST_EXP = -100


def quant_fp8_rows(x):
    """Rows of the 8-bit cache: (e4m3 codes of x's shape, exponent bytes uint8 of x's shape without the last dimension) with
    ``x ~ code * 2^(byte - 127)``. The exponent is the smallest one, but not under -100, with which the largest finite magnitude of a row is
    at most 448; codes are the nearest e4m3 numbers, ties to even; what is not finite is held as NaN. In 64 bits throughout."""
    xf = x.double()
    fine = torch.isfinite(xf)
    amax = torch.where(fine, xf.abs(), torch.zeros_like(xf)).amax(-1)
    frac, e = torch.frexp((amax / FP8_MAX).clamp_min(1e-200))         # amax / 448 = frac * 2^e, frac in [0.5, 1)
    e = torch.where(frac == 0.5, e - 1, e).clamp_min(FP8_ROW_LEAST_EXP)
    y = xf * _pow2_f64(-e).unsqueeze(-1)
    step = _pow2_f64((torch.frexp(y)[1] - 4).clamp_min(-9))           # distance of e4m3 numbers around y
    y = torch.where(fine, torch.round(y / step) * step, torch.full_like(y, math.nan))
    return y.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _pow2_f64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def dequant_fp8_rows(codes, scale_bytes, dtype=torch.float32):
    """Values of rows of the 8-bit cache (exact in fp32 and bf16)."""
    return (codes.double() * _pow2_f64(scale_bytes.long() - 127).unsqueeze(-1)).to(dtype)


def rope_kv_store_fp8(qkv, positions, slots, cos_sin, k_cache, v_cache, k_scale, v_scale, n_q, n_kv, head_dim, interleaved, rot_dims, q_out):
    T = qkv.shape[0]
    x = qkv[:, : (n_q + 2 * n_kv) * head_dim].reshape(T, n_q + 2 * n_kv, head_dim).double()
    if rot_dims:
        if bool(((positions[:T] < 0) | (positions[:T] >= cos_sin.shape[0])).any()):
            raise ValueError(f"a position out of [0, {cos_sin.shape[0]})")
        cs = cos_sin[positions[:T].long()].double().unsqueeze(1)
        c, s = cs[..., : rot_dims // 2], cs[..., rot_dims // 2:]
        turn = x[:, : n_q + n_kv, :rot_dims]
        if interleaved:
            a, b = turn[..., 0::2].clone(), turn[..., 1::2].clone()
            turn[..., 0::2], turn[..., 1::2] = a * c - b * s, b * c + a * s
        else:
            a, b = turn[..., : rot_dims // 2].clone(), turn[..., rot_dims // 2:].clone()
            turn[..., : rot_dims // 2], turn[..., rot_dims // 2:] = a * c - b * s, b * c + a * s
    q_out[:T, : n_q * head_dim] = x[:, :n_q].reshape(T, n_q * head_dim).to(qkv.dtype)
    page = k_cache.shape[2]
    if bool((slots[:T] >= k_cache.shape[0] * page).any()):
        raise ValueError(f"a slot past the {k_cache.shape[0] * page} of the cache")
    ok = slots[:T] >= 0
    pg, off = slots[:T][ok] // page, slots[:T][ok] % page
    for part, cache, scale in ((x[:, n_q: n_q + n_kv], k_cache, k_scale), (x[:, n_q + n_kv:], v_cache, v_scale)):
        codes, e = quant_fp8_rows(part[ok])
        cache.view(torch.uint8)[pg, :, off] = codes.view(torch.uint8)
        scale[pg, :, off] = e


def _fp8_rows_of(cache, scale, pages, n, dtype):
    """Rows [0, n) of a sequence: [n, heads, head_dim]."""
    need = -(-n // cache.shape[2])
    pages = pages[:need].long()
    if len(pages) < need or bool(((pages < 0) | (pages >= cache.shape[0])).any()):
        raise ValueError(f"{n} tokens on pages {pages.tolist()} of {cache.shape[0]}")
    v = dequant_fp8_rows(cache.view(torch.uint8)[pages].view(torch.float8_e4m3fn), scale[pages], dtype)
    return v.transpose(1, 2).reshape(-1, cache.shape[1], cache.shape[3])[:n]


def kv_load_fp8(k_cache, v_cache, k_scale, v_scale, block_table, kv_start, kv_len, k_out, v_out, rows):
    for out, cache, scale in ((k_out, k_cache, k_scale), (v_out, v_cache, v_scale)):
        out[:rows] = 0
        for s in range(block_table.shape[0]):
            a, n = int(kv_start[s]), int(kv_len[s])
            if n > 0:
                out[a: min(a + n, rows)] = _fp8_rows_of(cache, scale, block_table[s], n, out.dtype)[: max(0, rows - a)]


def paged_attention_fp8(q, k_cache, v_cache, k_scale, v_scale, block_table, q_start, q_len, kv_len, n_q, n_kv, head_dim, scale, out):
    for s in range(block_table.shape[0]):
        qs, ql, kl = int(q_start[s]), int(q_len[s]), int(kv_len[s])
        if ql <= 0:
            continue
        o = torch.zeros(ql, n_q, head_dim, dtype=torch.float32, device=q.device)
        if kl > 0:
            k, v = (_fp8_rows_of(c, e, block_table[s], kl, torch.float32).repeat_interleave(n_q // n_kv, 1)
                    for c, e in ((k_cache, k_scale), (v_cache, v_scale)))
            qq = q[qs: qs + ql, : n_q * head_dim].float().view(ql, n_q, head_dim)
            hidden = torch.arange(kl, device=q.device).unsqueeze(0) > torch.arange(kl - ql, kl, device=q.device).unsqueeze(1)
            w = torch.einsum("qhd,khd->hqk", qq, k).mul(scale).masked_fill(hidden, float("-inf"))
            w = torch.exp(w - w.amax(-1, keepdim=True).clamp_min(-1e30))
            bad = torch.isnan(v)                                                                       # (zero times NaN would reach rows that do not see it)
            o = torch.einsum("hqk,khd->qhd", w, v.masked_fill(bad, 0)) / w.sum(-1).t().unsqueeze(-1).clamp_min(1e-37)      # (rows without keys: zero)
            if bool(bad.any()):
                o.masked_fill_(torch.einsum("qk,khd->qhd", (~hidden).float(), bad.float()) > 0, math.nan)
        out[qs: qs + ql, : n_q * head_dim] = o.reshape(ql, -1).to(out.dtype)


# ---------------------------------------------------------------------- multi-head latent attention
def mla_kv_store(c_kv, k_rope, slots, cache):
    """Scatter one latent row per token: cache[page, offset] = [c_kv (kv_lora_rank) | k_rope].

    cache: [pages, page_size, kv_lora_rank + rope_dim] view of one layer; slots < 0 are skipped.
    """
    page_size = cache.shape[1]
    ok = slots >= 0
    pg = torch.div(slots.clamp(min=0), page_size, rounding_mode="floor")
    off = slots.clamp(min=0) % page_size
    row = torch.cat((c_kv, k_rope), dim=-1).to(cache.dtype)
    cache[pg[ok], off[ok]] = row[ok]


def mla_paged_attention(q_lat, q_rope, cache, block_table, q_start, q_len, kv_len, scale):
    """Absorbed-form MLA over the latent cache (one shared "KV head" for all query heads).

    q_lat: [T, h, R] queries already multiplied by W_uk; q_rope: [T, h, Dr] rotated;
    cache: [pages, page_size, R + Dr]. Returns the attention output in latent space [T, h, R]
    (the caller multiplies by W_uv).
    """
    T, h, R = q_lat.shape
    out = torch.zeros(T, h, R, dtype=q_lat.dtype, device=q_lat.device)
    page_size = cache.shape[1]
    for b in range(block_table.shape[0]):
        qs, ql, kl = int(q_start[b]), int(q_len[b]), int(kv_len[b])
        if ql == 0:
            continue
        n_pages = (kl + page_size - 1) // page_size
        kv = cache[block_table[b, :n_pages].long()].reshape(-1, cache.shape[-1])[:kl].float()
        c, kr = kv[:, :R], kv[:, R:]
        s = (torch.einsum("qhr,kr->hqk", q_lat[qs:qs + ql].float(), c) +
             torch.einsum("qhd,kd->hqk", q_rope[qs:qs + ql].float(), kr)) * scale
        qi = torch.arange(ql, device=s.device).unsqueeze(1) + (kl - ql)
        ki = torch.arange(kl, device=s.device).unsqueeze(0)
        p = torch.softmax(s.masked_fill(ki > qi, float("-inf")), dim=-1)
        out[qs:qs + ql] = torch.einsum("hqk,kr->qhr", p, c).to(out.dtype)
    return out


def batched_linear(x, w):
    """x: [B, M, K], w: [B, N, K] -> [B, M, N] (per-batch ``x @ w.T``)."""
    return torch.einsum("bmk,bnk->bmn", x.float(), w.float()).to(x.dtype)
