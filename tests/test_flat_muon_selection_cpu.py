"""Which parameters FlatMuon orthogonalises, over the framework's models."""

import pytest
import torch
import torch.nn as nn

from mvp_engine.models.qwen3 import build_qwen3
from mvp_engine.models.qwen3_vl import build_qwen3_vl
from mvp_engine.models.vit import build_vit
from mvp_engine.parallel.fsdp import NativeFSDP
from mvp_engine.parallel.optim import FlatMuon
from recipes.magic_transformer.model.magic_transformer import MagicTransformer, TransformerConfig


class OwnNames(nn.Module):
    """A model whose embedding's name says nothing; its head is tied to it."""

    def __init__(self):
        super().__init__()
        self.out = nn.Linear(8, 24, bias=False)
        self.wte = nn.Embedding(24, 8)
        self.out.weight = self.wte.weight
        self.mix = nn.Linear(8, 8)


MODELS = {
    "qwen3": (lambda: build_qwen3("mvp/qwen3-tiny", seed=3), {"model.embed_tokens.weight", "lm_head.weight"}),
    "qwen3 tied": (lambda: build_qwen3("mvp/qwen3-tiny", seed=3, tie_word_embeddings=True),
                   {"model.embed_tokens.weight", "lm_head.weight"}),
    "qwen3_vl": (lambda: build_qwen3_vl("mvp/qwen3-vl-tiny", seed=3),
                 {"model.language_model.embed_tokens.weight", "model.visual.pos_embed.weight", "lm_head.weight"}),
    "vit": (lambda: build_vit("vit-tiny-patch16-224", seed=3, num_hidden_layers=2, num_labels=10), {"classifier.weight"}),
    "magic": (lambda: MagicTransformer(TransformerConfig(vocab_size=64, d_model=32, n_layers=2)),
              {"embed.weight", "lm_head.weight"}),
    "own": (OwnNames, {"wte.weight", "out.weight"}),
}


@pytest.mark.parametrize("name", list(MODELS))
def test_embeddings_and_heads_are_left_to_adamw(name):
    make, kept_out = MODELS[name]
    model = make()
    matrices = {n for n, p in model.named_parameters(remove_duplicate=False) if p.dim() == 2}
    assert kept_out <= matrices
    fsdp = NativeFSDP(model, group=None, device=torch.device("cpu"), param_dtype=torch.float32)
    opt = FlatMuon(fsdp, lr=1e-3)
    taken = {f for es in opt._matrices.values() for e in es for f in e.fqns}
    assert taken == matrices - kept_out and taken
    chosen = FlatMuon(fsdp, lr=1e-3, matrix_filter=lambda fqn, shape: fqn in kept_out)
    assert {e.fqns[0] for es in chosen._matrices.values() for e in es} <= kept_out
