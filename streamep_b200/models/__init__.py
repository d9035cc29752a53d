"""Model-side pieces: the ``StreamMoE`` module, a small language model with its optimizer, and the pure-PyTorch oracles."""
import importlib


def __getattr__(name):
    if name in ("StreamMoE", "make_buffer"):
        return getattr(importlib.import_module(__name__ + ".moe_layer"), name)
    if name in ("MoELM", "ExpertAdamW"):
        return getattr(importlib.import_module(__name__ + ".moe_lm"), name)
    raise AttributeError(name)
