"""The GPT's logits in float64 with keys and values as an 8-bit cache holds them, and what speculative decoding has to
answer with: the definition, without caches, chunks or a draft."""
import numpy as np
import torch

import chunk_helpers as ch
import torch_gpt


def held(x, dk, bits):
    """Keys or values (D, T) as a cache holds them: per position and head of dk rows."""
    if bits == 32:
        return x
    by, scale = ch.quantise(x.numpy().T.reshape(-1, dk))
    return torch.as_tensor((by * scale[:, None].astype(np.float64)).reshape(x.shape[1], -1).T.copy())


def logits(params_np, seq, cfg, bits=32):
    """(T, vocab) of one sequence."""
    T, D, H, F = len(seq), cfg["d_model"], cfg["num_heads"], cfg["d_ff"]
    dk, pos = D // H, cfg["pos_enc"]
    it = iter([torch.as_tensor(np.asarray(p, np.float64)) for p in params_np])
    x = next(it)[torch.as_tensor(np.asarray(seq, np.int64))]
    if pos == "learned":
        x = x + next(it)[:T]
    elif pos == "sinusoidal":
        x = x + torch_gpt._sinusoidal(T, D)
    x = x.T

    def norm(x):
        if cfg.get("norm") == "layernorm":
            g, b = next(it), next(it)
            return torch_gpt._layernorm(x, g, b)
        return torch_gpt._rmsnorm(x, next(it))

    for _ in range(cfg["num_layers"]):
        Wq, bq, Wk, bk, Wv, bv, Wo, bo = (next(it) for _ in range(8))
        h = norm(x)
        q, k, v = Wq @ h + bq, Wk @ h + bk, Wv @ h + bv
        if pos == "rope":
            q, k = (torch.cat([torch_gpt._rope(z[i:i + dk], T, dk) for i in range(0, D, dk)]) for z in (q, k))
        k, v = held(k, dk, bits), held(v, dk, bits)
        out = torch.zeros_like(q)
        for hh in range(H):
            r = slice(hh * dk, (hh + 1) * dk)
            S = q[r].T @ k[r] / np.sqrt(dk) + torch_gpt._mask(T, hh, H, pos == "alibi", None)
            out[r] = v[r] @ torch.softmax(S, dim=1).T
        x = x + (Wo @ out + bo)
        W1, b1, W2, b2 = (next(it) for _ in range(4))
        u = W1 @ norm(x) + b1
        if cfg.get("activation", "swiglu") == "swiglu":
            act = u[:F] * torch.sigmoid(u[:F]) * u[F:]
        else:
            act = u * torch.sigmoid(1.702 * u)
        x = x + (W2 @ act + b2)
    g = norm(x)
    W, b = next(it), next(it)
    return (W @ g + b).T.numpy()


def limit(cfg, prompt, max_new):
    return min(max_new, cfg["seq_len"] - len(prompt) + 1)


def check_greedy(found, params, prompt, max_new, eos, cfg, bits, gap):
    """Each token has the largest logit behind its predecessors, or one that lies at most `gap` below it; the sequence ends
    where it has to. Returns how many were decided by more than the gap."""
    steps = limit(cfg, prompt, max_new)
    assert len(found) <= steps and eos not in found
    rows = found + ([eos] if len(found) < steps else [])
    clear = 0
    for i, t in enumerate(rows):
        z = logits(params, list(prompt) + rows[:i], cfg, bits)[-1]
        assert z[t] >= z.max() - gap, (i, t)
        clear += int(np.sort(z)[-1] - np.sort(z)[-2] > gap) if len(z) > 1 else 1
    return clear
