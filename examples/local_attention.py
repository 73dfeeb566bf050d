"""One decoder layer's local attention, trained and then served.

    python examples/local_attention.py

Training: a packed q, k, v projection (kda.matmul's product stands for the
model's), per-head norms with the position rotation, attention inside a sliding
window with sinks, and the gradients of all of it.  Serving: a ragged batch of
prompts goes into the key/value cache, then tokens are decoded one by one; the
decode's rows are compared with the rows of the training forward.
"""

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "kda-for-trainium_b200"))
import kda  # noqa: E402
import kda.autograd as ka  # noqa: E402

B, S, MODEL, QH, KH, D = 4, 600, 1024, 16, 4, 128
WINDOW, SINKS = 256, 4


def main():
    torch.manual_seed(0)
    dev, bf16 = "cuda", torch.bfloat16
    w = (torch.randn(MODEL, (QH + 2 * KH) * D, device=dev) * MODEL ** -0.5).to(bf16)
    gq = torch.ones(D, device=dev, requires_grad=True)
    gk = torch.ones(D, device=dev, requires_grad=True)
    table = kda.rope_table(S, D, 10000.0)  # kept with the model
    x = torch.randn(B * S, MODEL, device=dev).to(bf16)

    # one training step's forward and backward
    qkv = kda.matmul(x, w).view(B, S, -1).requires_grad_()
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split((QH * D, KH * D, KH * D), dim=-1))
    qr, kr = ka.qk_norm_rope(q, k, gq, gk, table)
    out = ka.gqa_window(qr, kr, v, WINDOW, SINKS)
    loss = out.float().square().mean()
    loss.backward()
    print(f"loss {loss.item():.6f}  |dqkv| {qkv.grad.float().norm().item():.4e}  |dgq| {gq.grad.norm().item():.4e}")

    # serving: prompts of different lengths, slot 3 idle
    prompt = torch.tensor([500, 17, 333, -1], dtype=torch.int32, device=dev)
    k_cache = torch.zeros(B, S, KH, D, dtype=bf16, device=dev)
    v_cache = torch.zeros_like(k_cache)
    worst = 0.0
    with torch.no_grad():
        for b, n in enumerate(prompt.tolist()):  # each prompt into its slot of the cache
            if n > 0:
                zero = torch.zeros(1, dtype=torch.int32, device=dev)
                kda.qk_norm_rope_append(q[b:b + 1, :n], k[b:b + 1, :n], v[b:b + 1, :n], gq, gk, table,
                                        k_cache[b:b + 1], v_cache[b:b + 1], zero)
        n = prompt.clone()
        rows = torch.arange(B, device=dev)
        for _ in range(20):
            at = n.clamp(min=0).long()
            step = [t[rows, at].unsqueeze(1).contiguous() for t in (q, k, v)]  # this step's token of each slot
            qs = kda.qk_norm_rope_append(*step, gq, gk, table, k_cache, v_cache, n)
            n = torch.where(n >= 0, n + 1, n)
            y = kda.gqa_window_decode(qs[:, 0], k_cache, v_cache, n, WINDOW, SINKS)
            live = n > 0
            want = out[rows, at]
            err = (y[live].float() - want[live].float()).norm() / want[live].float().norm()
            worst = max(worst, err.item())
            assert not y[~live].any()
    torch.cuda.synchronize()
    assert kda.device_error() == 0
    print(f"20 decoded tokens: rows within {worst:.2e} of the forward's")
    return worst


if __name__ == "__main__":
    # the two sides round the softmax weights and the result to bf16 each: 4 x 2^-8 at most
    assert main() <= 4 * 2.0 ** -8
