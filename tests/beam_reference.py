"""Beam search in float64 over torch_gpt's forward: the definition, without caches or tables."""
import numpy as np
import torch

import torch_gpt


def log_probs(params, seqs, cfg):
    """Log probabilities (n, vocab) of the token after each of n sequences of one length."""
    tokens = torch.as_tensor(np.array(seqs).T)
    T = tokens.shape[0]
    if cfg["pos_enc"] == "learned":   # the model of a context of T: the first T positions
        params = [params[0], params[1][:T]] + list(params[2:])
    with torch.no_grad():
        logits = torch_gpt.forward(params, tokens, dict(cfg, seq_len=T))
    return torch.log_softmax(logits[:, T - 1::T].T, dim=1).numpy()


def total(params, prompt, tokens, eos, cfg):
    """Sum of log probabilities of a continuation (eos appended where given)."""
    seq, s = list(prompt), 0.0
    for t in list(tokens) + ([] if eos is None else [eos]):
        s += log_probs(params, [seq], cfg)[0, t]
        seq.append(t)
    return s


def beam_search(params_np, prompt, beams, max_new, eos, cfg):
    """[(tokens without eos, total, ended)] best first, and the smallest gap between totals that were compared."""
    params = [torch.as_tensor(np.asarray(p, np.float64)) for p in params_np]
    steps = min(max_new, cfg["seq_len"] - len(prompt) + 1)
    live, gap, V = [([], 0.0, False)], np.inf, cfg["vocab_size"]
    for _ in range(steps):
        cand = []
        going = [i for i, x in enumerate(live) if not x[2]]
        lp = log_probs(params, [list(prompt) + live[i][0] for i in going], cfg) if going else None
        for i, (toks, score, ended) in enumerate(live):
            if ended:
                cand.append((score, i * V + eos, toks, True))
            else:
                row = score + lp[going.index(i)]
                for v in np.argsort(-row)[:beams + 1]:
                    cand.append((row[v], i * V + v, toks + ([] if v == eos else [int(v)]), v == eos))
        cand.sort(key=lambda c: (-c[0], c[1]))
        s = np.array([c[0] for c in cand[:beams + 1]])
        if len(s) > 1:
            gap = min(gap, float((s[:-1] - s[1:]).min()))
        live = [(t, sc, e) for sc, _, t, e in cand[:beams]]
        if all(x[2] for x in live):
            break
    return live, gap
