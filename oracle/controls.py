"""Penalties, biases and token masks on logits in float64 with numpy: what
sampling.LogitControls computes, row by row and token by token."""
import numpy as np


def control_rows(logits, history, lengths, prompts, counts, proposed, *, repetition, presence, frequency, bias, allowed,
                 fill, lowest, slots=None):
    """float64 rows.  logits float64 [rows, V]; history int [texts, capacity]; allowed
    bool [rows, V] or None; lowest, highest finite value of the output: +-lowest."""
    logits = np.asarray(logits, np.float64)
    out = np.empty_like(logits)
    v, row, at = logits.shape[1], 0, 0
    for r, n in enumerate(counts):
        text = list(history[r if slots is None else slots[r]][:lengths[r]])
        for j in range(n + 1):
            answer = [int(t) for t in text[prompts[r]:] + list(proposed[at:at + j]) if 0 <= t < v]
            seen = set(answer) | {int(t) for t in text[:prompts[r]] if 0 <= t < v}
            y = logits[row].copy()
            with np.errstate(invalid='ignore', over='ignore'):
                for t in seen:
                    y[t] = y[t] / repetition[r] if y[t] > 0 else y[t] * repetition[r]
                for t in set(answer):
                    y[t] -= answer.count(t) * frequency[r] + presence[r]
                for t, b in (bias[r] or {}).items():
                    y[t] += b
            finite = np.isfinite(logits[row])
            y[finite] = np.clip(y[finite], lowest, -lowest)
            if allowed is not None:
                y[~allowed[row]] = fill if allowed[row].any() else -np.inf
            out[row] = y
            row += 1
        at += n
    return out
