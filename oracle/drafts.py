"""Plain restatement of the verification of drafted tokens
(include/epure_draft.h), one sequence and token after the other in Python's
floats (64 bits).  Pinned by tests/test_drafts_cpu.py, which counts outcomes."""
import torch


def verify(target, drafted, uniforms, draft=None):
    """(accepted, tokens) as lists.  A probability that is negative or no number is 0."""
    target, drafted, uniforms = target.detach().cpu().double(), drafted.cpu().tolist(), uniforms.cpu().double().tolist()
    draft = None if draft is None else draft.detach().cpu().double()
    target = torch.where(target > 0, target, 0.0)
    draft = None if draft is None else torch.where(draft > 0, draft, 0.0)
    B, n, V = len(drafted), target.shape[1] - 1, target.shape[2]
    accepted, tokens = [], []
    for b in range(B):
        k, down = 0, False
        for i in range(n):
            x = drafted[b][i]
            if not 0 <= x < V:
                break
            q = 1.0 if draft is None else draft[b, i, x].item()
            if not uniforms[b][i] * q < target[b, i, x].item():
                down = True
                break
            k += 1
        p = target[b, k].tolist()
        if not down:
            r = p
        elif draft is None:
            r = [w - (1.0 if v == drafted[b][k] else 0.0) for v, w in enumerate(p)]
        else:
            r = [w - z for w, z in zip(p, draft[b, k].tolist())]
        r = [w if w > 0 else 0.0 for w in r]
        if not any(r):
            r = p
        goal, run, pick = uniforms[b][n] * sum(r), 0.0, V - 1
        some = [v for v, w in enumerate(r) if w > 0]
        if some:
            pick = some[-1]
            for v in some:
                run += r[v]
                if run > goal:
                    pick = v
                    break
        accepted.append(k)
        tokens.append(drafted[b][:k] + [pick] + [-1] * (n - k))
    return accepted, tokens
