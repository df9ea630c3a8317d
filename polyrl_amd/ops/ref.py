"""Pure-PyTorch reference implementations of every HIP kernel.

These are the numerics oracles: each HIP kernel in csrc/ is tested against the
fp32 form here (tests/test_ops_gpu.py), and they serve as the CPU execution
path for the no-GPU test tier.  Keep them simple and obviously correct.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    xf = x.float()
    var = xf.pow(2).mean(-1, keepdim=True)
    out = xf * torch.rsqrt(var + eps) * weight.float()
    return out.to(x.dtype)


def fused_add_rmsnorm(x: torch.Tensor, residual: torch.Tensor,
                      weight: torch.Tensor, eps: float = 1e-6
                      ) -> Tuple[torch.Tensor, torch.Tensor]:
    """returns (rmsnorm(x + residual), x + residual)"""
    new_residual = (x.float() + residual.float()).to(x.dtype)
    return rmsnorm(new_residual, weight, eps), new_residual


def rope_cos_sin(positions: torch.Tensor, head_dim: int, theta: float = 10000.0,
                 dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos/sin tables for given positions. (N,) -> (N, head_dim//2)."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2,
                                             device=positions.device).float() / head_dim))
    freqs = positions.float().unsqueeze(-1) * inv_freq  # (N, D/2)
    return freqs.cos().to(dtype), freqs.sin().to(dtype)


def apply_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor,
               sin: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """NEOX-style (rotate-half) RoPE.

    q: (N, Hq, D), k: (N, Hk, D); cos/sin: (N, D/2).
    """
    def rot(x):
        d = x.shape[-1] // 2
        x1, x2 = x[..., :d], x[..., d:]
        c = cos.unsqueeze(1)  # (N,1,D/2)
        s = sin.unsqueeze(1)
        o1 = x1.float() * c - x2.float() * s
        o2 = x2.float() * c + x1.float() * s
        return torch.cat([o1, o2], dim=-1).to(x.dtype)
    return rot(q), rot(k)


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    return (torch.nn.functional.silu(gate.float()) * up.float()).to(gate.dtype)


def gather_logprobs(logits: torch.Tensor, labels: torch.Tensor
                    ) -> torch.Tensor:
    """(N, V), (N,) -> (N,) log softmax at labels, fp32."""
    logp = torch.log_softmax(logits.float(), dim=-1)
    return torch.gather(logp, -1, labels.unsqueeze(-1)).squeeze(-1)


def gather_logprobs_entropy(logits: torch.Tensor, labels: torch.Tensor
                            ) -> Tuple[torch.Tensor, torch.Tensor]:
    logp = torch.log_softmax(logits.float(), dim=-1)
    lp = torch.gather(logp, -1, labels.unsqueeze(-1)).squeeze(-1)
    # a banned token (-inf) has no part in the entropy: 0, not 0 * inf
    low = torch.finfo(logp.dtype).min
    ent = -(logp.exp() * logp.clamp_min(low)).sum(-1)
    return lp, ent


def top_k_top_p_sample(logits: torch.Tensor, temperature: torch.Tensor,
                       top_k: torch.Tensor, top_p: torch.Tensor,
                       generator: Optional[torch.Generator] = None
                       ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-row temperature + top-k + top-p filtering and categorical draw.

    logits (N, V) fp32; temperature/top_k/top_p per-row (N,).
    Returns (token_ids (N,) int64, logprobs (N,) fp32 of the sampled token
    under the *filtered, renormalized* distribution's log-softmax of the
    ORIGINAL distribution — we report logprob under the unfiltered softmax,
    matching what rollout clients consume as output_token_logprobs).
    greedy when temperature == 0.
    """
    N, V = logits.shape
    logits = logits.float()
    out_tokens = torch.empty(N, dtype=torch.long, device=logits.device)
    logp_full = torch.log_softmax(logits, dim=-1)
    for i in range(N):
        t = float(temperature[i])
        if t == 0.0:
            tok = int(torch.argmax(logits[i]).item())
            out_tokens[i] = tok
            continue
        row = logits[i] / t
        k = int(top_k[i])
        if 0 < k < V:
            kth = torch.topk(row, k).values[-1]
            row = torch.where(row < kth, torch.full_like(row, float("-inf")), row)
        p = float(top_p[i])
        if p < 1.0:
            sorted_row, idx = torch.sort(row, descending=True)
            probs = torch.softmax(sorted_row, dim=-1)
            cum = torch.cumsum(probs, dim=-1)
            # keep tokens until cumulative prob exceeds p (always keep first)
            cutoff = cum - probs >= p
            sorted_row[cutoff] = float("-inf")
            row = torch.full_like(row, float("-inf"))
            row[idx] = sorted_row
        probs = torch.softmax(row, dim=-1)
        tok = int(torch.multinomial(probs, 1, generator=generator).item())
        out_tokens[i] = tok
    logps = logp_full.gather(-1, out_tokens.unsqueeze(-1)).squeeze(-1)
    return out_tokens, logps


def paged_attention_decode(
    q: torch.Tensor,            # (B, Hq, D)
    kv_cache_k: torch.Tensor,   # (num_pages, page_size, Hk, D)
    kv_cache_v: torch.Tensor,   # (num_pages, page_size, Hk, D)
    page_table: torch.Tensor,   # (B, max_pages) int32
    context_lens: torch.Tensor, # (B,) int32  (length INCLUDING current token)
    scale: float,
) -> torch.Tensor:
    """One new query token per sequence attending to its paged KV history."""
    B, Hq, D = q.shape
    Hk = kv_cache_k.shape[2]
    page_size = kv_cache_k.shape[1]
    g = Hq // Hk
    out = torch.empty_like(q, dtype=torch.float32)
    for b in range(B):
        L = int(context_lens[b])
        n_pages = -(-L // page_size)
        pages = page_table[b, :n_pages].long()
        k = kv_cache_k[pages].reshape(-1, Hk, D)[:L].float()  # (L, Hk, D)
        v = kv_cache_v[pages].reshape(-1, Hk, D)[:L].float()
        for h in range(Hq):
            hk = h // g
            s = (q[b, h].float() @ k[:, hk].T) * scale       # (L,)
            p = torch.softmax(s, dim=-1)
            out[b, h] = p @ v[:, hk]
    return out.to(q.dtype)


def varlen_prefill_attention(
    q: torch.Tensor,            # (total_q, Hq, D)
    k: torch.Tensor,            # (total_k, Hk, D)
    v: torch.Tensor,            # (total_k, Hk, D)
    cu_seqlens_q: torch.Tensor, # (B+1,)
    cu_seqlens_k: torch.Tensor, # (B+1,)
    scale: float,
    causal: bool = True,
) -> torch.Tensor:
    """Varlen (packed) causal attention.  When seqlen_k > seqlen_q the query
    block is aligned to the END of the keys (chunked-prefill semantics)."""
    Hq, D = q.shape[1], q.shape[2]
    Hk = k.shape[1]
    g = Hq // Hk
    out = torch.empty_like(q, dtype=torch.float32)
    B = cu_seqlens_q.shape[0] - 1
    for b in range(B):
        q0, q1 = int(cu_seqlens_q[b]), int(cu_seqlens_q[b + 1])
        k0, k1 = int(cu_seqlens_k[b]), int(cu_seqlens_k[b + 1])
        Lq, Lk = q1 - q0, k1 - k0
        qi = q[q0:q1].float()
        ki = k[k0:k1].float()
        vi = v[k0:k1].float()
        for h in range(Hq):
            hk = h // g
            s = (qi[:, h] @ ki[:, hk].T) * scale  # (Lq, Lk)
            if causal:
                qpos = torch.arange(Lq, device=q.device).unsqueeze(1) + (Lk - Lq)
                kpos = torch.arange(Lk, device=q.device).unsqueeze(0)
                s = s.masked_fill(kpos > qpos, float("-inf"))
            p = torch.softmax(s, dim=-1)
            out[q0:q1, h] = p @ vi[:, hk]
    return out.to(q.dtype)


def varlen_lse(q, k, cu_seqlens_q, cu_seqlens_k, scale, causal=True):
    """Log-sum-exp of the (masked) attention scores per (token, q-head) —
    reference for the prefill kernel's LSE output."""
    Hq = q.shape[1]
    Hk = k.shape[1]
    g = Hq // Hk
    out = torch.empty(q.shape[0], Hq, dtype=torch.float32)
    B = cu_seqlens_q.shape[0] - 1
    for b in range(B):
        q0, q1 = int(cu_seqlens_q[b]), int(cu_seqlens_q[b + 1])
        k0, k1 = int(cu_seqlens_k[b]), int(cu_seqlens_k[b + 1])
        Lq, Lk = q1 - q0, k1 - k0
        qi = q[q0:q1].float()
        ki = k[k0:k1].float()
        for h in range(Hq):
            s = (qi[:, h] @ ki[:, h // g].T) * scale
            if causal:
                qpos = torch.arange(Lq).unsqueeze(1) + (Lk - Lq)
                kpos = torch.arange(Lk).unsqueeze(0)
                s = s.masked_fill(kpos > qpos, float("-inf"))
            out[q0:q1, h] = torch.logsumexp(s, dim=-1)
    return out


def rows_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two operands share memory: rows of adjacent numbers (N, W) that may lie
    apart, or contiguous tensors.  The rule of rows_overlap.h."""
    def rows(t):
        size = t.element_size()
        if t.dim() != 2 or t.numel() == 0 or t.shape[0] == 1:
            return t.data_ptr(), 1, 0, t.numel() * size
        return t.data_ptr(), t.shape[0], t.stride(0) * size, t.shape[1] * size
    p, q = rows(a), rows(b)
    ends = [at + (n - 1) * pitch + width for at, n, pitch, width in (p, q)]
    if not p[3] or not q[3] or ends[0] <= q[0] or ends[1] <= p[0]:
        return False
    if p[2] == q[2] == 0:
        return True
    (at0, n0, pitch0, w0), (at1, n1, pitch1, w1) = (q, p) if q[2] == 0 else (p, q)
    same = pitch0 == pitch1
    for i in range(1 if same else n0):
        d = at0 + i * pitch0 - at1
        low, high = (d - w1) // pitch1 + 1, -(-(d + w0) // pitch1) - 1
        if max(low, 1 - n0 if same else 0) <= min(high, n1 - 1):
            return True
    return False


# ------------------------------------------------------- adapters of requests


def adapter_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor,
                b: torch.Tensor, scale: torch.Tensor, index: torch.Tensor,
                widths, ranks: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y + scale[i] * B_i (A_i x) by every row's adapter i = index[t]; rows without one
    are y's.  a (S, P, r, K), b (S, N, r), parts of ``widths`` columns."""
    S, P, r, K = a.shape
    if (x.shape != (y.shape[0], K) or b.shape != (S, y.shape[1], r)
            or len(widths) != P or sum(widths) != y.shape[1]):
        raise ValueError("adapter_add: shapes that do not fit together")
    out = y.clone()
    for s in range(S):
        rows = (index == s).nonzero().flatten()
        n = r if ranks is None else min(max(int(ranks[s]), 0), r)
        if not len(rows) or n == 0:
            continue
        total = y[rows].float()
        at = 0
        for p, w in enumerate(widths):
            h = x[rows].float() @ a[s, p, :n].float().t() * scale[s]
            total[:, at:at + w] += h @ b[s, at:at + w, :n].float().t()
            at += w
        out[rows] = total.to(y.dtype)
    return out


# ------------------------------------------------------------ rules on logits


def adjust_logits(logits: torch.Tensor, rules, rows: torch.Tensor
                  ) -> torch.Tensor:
    out = logits.clone()
    V = logits.shape[1]
    for i, s in enumerate(rows.tolist()):
        if not 0 <= s < rules.slots:
            continue
        total = min(max(int(rules.total_len[s]), 0), rules.capacity)
        prompt = min(max(int(rules.prompt_len[s]), 0), total)
        words = rules.history[s, :total].long()
        known = (words >= 0) & (words < V)
        asked, said = (torch.bincount(w[k], minlength=V) for w, k in (
            (words[:prompt], known[:prompt]), (words[prompt:], known[prompt:])))
        x = logits[i].float()
        rep = rules.repetition[s]
        x = torch.where(asked + said > 0, torch.where(x > 0, x / rep, x * rep), x)
        x = torch.where(said > 0, x - rules.frequency[s] * said.float()
                        - rules.presence[s], x)
        last = {t: v for t, v in zip(rules.bias_tokens[s].tolist(),
                                     rules.bias_values[s].tolist())
                if 0 <= t < V}
        if last:
            x[list(last)] += torch.tensor(list(last.values()))
        if rules.masked[s]:
            words = rules.mask[s].unsqueeze(1) >> torch.arange(32)
            x = x.masked_fill((words & 1).flatten()[:V] == 0, float("-inf"))
        out[i] = x.to(logits.dtype)
    return out


def append_tokens(rules, rows: torch.Tensor, tokens: torch.Tensor) -> None:
    for s, t in zip(rows.tolist(), tokens.tolist()):
        if not 0 <= s < rules.slots:
            continue
        at = max(int(rules.total_len[s]), 0)
        if at < rules.capacity:
            rules.history[s, at] = t if 0 <= t < 1 << 31 else -1
            rules.total_len[s] = at + 1


# ------------------------------------------------------------- seeded dropout


def dropout_keep(numel: int, drop: int, seed: int) -> torch.Tensor:
    """Whether each of ``numel`` elements stays: Philox4x32-10 (Salmon, Moraes, Dror and
    Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011), eight numbers of 16
    bits for every counter, key = seed."""
    low = (1 << 32) - 1
    at = torch.arange((numel + 7) // 8)
    zero = torch.zeros_like(at)
    c = [at & low, at >> 32, zero, zero]
    key = [seed & low, (seed >> 32) & low]
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((q >> 32) & low) ^ c[1] ^ key[0], q & low,
             ((p >> 32) & low) ^ c[3] ^ key[1], p & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    words = torch.stack(c, -1)
    return torch.stack([words & 0xffff, words >> 16], -1).flatten()[:numel] >= drop


def dropout(x: torch.Tensor, drop: int, seed: torch.Tensor) -> torch.Tensor:
    """Elements that stay, times 65536 / (65536 - drop); zeros for the others."""
    keep = dropout_keep(x.numel(), drop, int(seed)).view(x.shape)
    scale = 65536.0 / (65536 - drop) if drop < 65536 else 0.0
    return torch.where(keep, x.float() * scale, 0.0).to(x.dtype)
