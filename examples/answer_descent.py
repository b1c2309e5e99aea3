"""Trains table rows and the PLE block's projections on answers: first on pairs
of a preferred and a rejected answer, then on sampled answers with a reward.

    python examples/answer_descent.py [steps]

A packed bin holds the fragments (prompt + answer); its positions' n-gram rows
are gathered and consumed by the PLE block, and a fixed head gives the logits.
The rows read by the answers are the variables (``DescentState``, Adam), the
block's key projection (a matrix a stream) and value projection are trained with
orthogonalised updates (``MuonState``).  The reference policy of both losses is
the same model before training, the table without overlay.  Everything is
synthetic and seeded."""
from __future__ import annotations

import sys
import types
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import __graft_entry__  # noqa: E402

__graft_entry__.load_package()

from engraft_ngram_amd import losses, muon, ple, synthetic  # noqa: E402
from engraft_ngram_amd.descent import DescentState  # noqa: E402
from engraft_ngram_amd.pack import pack_fragments, seg_starts_from_segment_ids  # noqa: E402

EOS, VOCAB, PROMPT = synthetic.QWEN_EOS, 4001, 12
STREAMS, DIM, HEADS = 4, 128, 16
WIDTH = DIM * HEADS  # n_embd: the gathered rows side by side
HPARAMS = types.SimpleNamespace(hc_mult=STREAMS, n_embd=WIDTH, f_norm_rms_eps=1e-6, ple_ngram_size=3)


class Answers:
    """One packed bin of fragments, the model around the table, and what trains."""

    def __init__(self, fragments: list[list[int]], seed: int):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def some(*shape, size):
            return torch.randn(shape, generator=g, device="cuda") * size

        bins = pack_fragments(fragments, EOS, max_len=4096)
        if len(bins) != 1:
            raise ValueError("the fragments must fit one bin")
        packed = bins[0]
        tokens = np.asarray(packed.tokens, dtype=np.int64)
        self.n = len(tokens) - 1
        self.tokens = torch.from_numpy(tokens[:self.n]).cuda()
        self.segment_ids = packed.segment_ids.cuda()
        self.seg_start = seg_starts_from_segment_ids(packed.segment_ids)
        # targets: the answers' tokens; prompts and the positions between fragments are left out
        targets = np.full(self.n, -100, dtype=np.int64)
        for start, end in packed.frag_slices:
            targets[start + PROMPT:end] = tokens[start + PROMPT + 1:end + 1]
        self.targets = torch.from_numpy(targets).cuda()
        self.n_segments = len(fragments)

        self.table = synthetic.table("q8_0", HEADS * 8192, DIM, seed=seed, hash_seed=seed + 1)
        self.rows = self.table.rows(self.tokens, seg_start=self.seg_start)
        self.state = DescentState.from_rows(self.table, self.rows, quant_fmt=None)
        self.weights = ple.PleWeights(
            w_key=some(STREAMS * WIDTH, WIDTH, size=WIDTH ** -0.5), w_value=some(WIDTH, WIDTH, size=WIDTH ** -0.5),
            norm_key=torch.ones(STREAMS * WIDTH, device="cuda"), norm_query=torch.ones(STREAMS * WIDTH, device="cuda"),
            norm_conv=torch.ones(STREAMS * WIDTH, device="cuda"), conv1d=some(STREAMS * WIDTH, 4, size=0.1))
        self.hidden = some(self.n, STREAMS, WIDTH, size=0.1)
        self.head = some(VOCAB, WIDTH, size=0.1)
        self.history = torch.zeros((0, STREAMS, WIDTH), device="cuda")
        w = self.weights
        self.optimizer = muon.MuonState([w.w_key.view(STREAMS, WIDTH, WIDTH), w.w_value])

    def embed(self, overlay: bool = True) -> torch.Tensor:
        """The positions' rows side by side, f32 ``[n, WIDTH]``: the variables where ``overlay``."""
        return self.table.forward(self.tokens, None, seg_start=self.seg_start,
                                  overlay=self.state.overlay(quantized=False) if overlay else None)

    def logits(self, emb: torch.Tensor) -> torch.Tensor:
        out, _ = ple.ple_forward(emb, self.hidden, self.weights, self.history, HPARAMS)
        return (out.mean(dim=1) @ self.head.T).to(torch.bfloat16)

    def step(self, loss_of, lr_rows: float, lr_weights: float):
        """One step of the rows and the projections on ``loss_of(logits)``."""
        w = self.weights
        emb = self.embed().requires_grad_()
        for p in (w.w_key, w.w_value):
            p.requires_grad_()
        result = loss_of(self.logits(emb))
        d_emb, d_key, d_value = torch.autograd.grad(result.loss, [emb, w.w_key, w.w_value])
        for p in (w.w_key, w.w_value):
            p.requires_grad_(False)
        self.state.step(d_emb, self.rows, lr=lr_rows, dense=True)
        self.optimizer.step([d_key.view(STREAMS, WIDTH, WIDTH), d_value], lr=lr_weights)
        return result


def run(steps: int = 8, pairs: int = 6, seed: int = 1) -> dict[str, list[float]]:
    """Losses (and the mean margin) before every step of both trainings."""
    rng = np.random.default_rng(seed)

    def fragment(prompt, length):
        return list(prompt) + rng.integers(10, VOCAB, length).tolist()

    prompts = [rng.integers(10, VOCAB, PROMPT) for _ in range(pairs)]
    fragments = [fragment(p, int(rng.integers(9, 40))) for p in prompts for _ in range(2)]  # chosen, rejected, ...
    model = Answers(fragments, seed)

    reference = losses.token_logprobs(model.logits(model.embed(overlay=False)), model.targets)
    sums = torch.zeros(model.n_segments, device="cuda").index_add_(0, model.segment_ids, reference)
    history = {"preference": [], "margin": [], "policy": []}
    for _ in range(steps):
        r = model.step(lambda z: losses.preference_loss(z, model.targets, model.segment_ids, sums, beta=0.1),
                       lr_rows=1e-4, lr_weights=1e-4)
        history["preference"].append(float(r.loss.detach()))
        history["margin"].append(float(r.margins.mean()))

    # sampled answers: a reward each, normalised over the bin; the policy that sampled them is today's
    reward = torch.from_numpy(rng.normal(size=model.n_segments).astype(np.float32)).cuda()
    advantages = ((reward - reward.mean()) / reward.std())[model.segment_ids]
    old = losses.token_logprobs(model.logits(model.embed()), model.targets)
    for _ in range(steps):
        r = model.step(lambda z: losses.policy_loss(z, model.targets, advantages, old, ref_logprobs=reference, kl_coef=0.01,
                                                    clip=(0.2, 0.28), segment_ids=model.segment_ids,
                                                    n_segments=model.n_segments, reduction="sequence"),
                       lr_rows=1e-4, lr_weights=1e-4)
        history["policy"].append(float(r.loss.detach()))
    return history


if __name__ == "__main__":
    for name, values in run(int(sys.argv[1]) if len(sys.argv) > 1 else 8).items():
        print(f"{name:10s} " + " ".join(f"{x:8.4f}" for x in values))
