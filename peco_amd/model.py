"""Installing PECO on a transformer (the peco/model.py interface: install_attention, reset_state); its attention
projections in 8 bits (quantize_projections).

An installation is one object kept on the transformer. It owns the shared
``InferenceContext``, one ``PecoAttention`` per attention block (double-stream blocks first,
then single-stream blocks, so a processor's index is its layer index) and the forward
pre-hook that refreshes the context before every transformer call. Installing again replaces
the previous installation: its hook is removed first, so a transformer never advances the
step twice per call.

Works with any pipeline whose ``transformer`` has ``transformer_blocks`` and
``single_transformer_blocks`` (blocks with ``attn.set_processor``) and a ``forward`` that
takes ``encoder_attention_mask`` (HunyuanVideo in diffusers).
"""
from __future__ import annotations

import inspect
from dataclasses import dataclass, field

import torch

from . import projection
from .processor import InferenceContext, PecoAttention, PecoConfig

_ATTRIBUTE = "_peco_installation"


def _text_lengths(mask):
    """(total, valid) text lengths of one prompt's right-padded mask [1, T].

    The reference's hook accepts exactly one prompt and masks whose valid tokens form a
    prefix (peco/model.py:25-34); the same errors are raised here.
    """
    if mask.shape[0] != 1:
        raise ValueError("Use one prompt per inference call")
    row = mask[0].detach().to(device="cpu", dtype=torch.bool)
    valid = int(row.sum())
    prefix = torch.arange(row.numel()) < valid
    if not torch.equal(row, prefix):
        raise ValueError("Hunyuan text attention mask must use right padding")
    return row.numel(), valid


@dataclass
class _Installation:
    context: InferenceContext
    processors: list
    signature: inspect.Signature
    handle: object = field(default=None)

    def before_forward(self, module, args, kwargs):
        """Forward pre-hook: one transformer call is one denoising step."""
        bound = self.signature.bind_partial(*args, **kwargs).arguments
        total, valid = _text_lengths(bound["encoder_attention_mask"])
        self.context.step += 1
        self.context.text_length = total
        self.context.valid_text_length = valid

    def reset(self):
        self.context.step = -1
        for processor in self.processors:
            processor.reset()

    def remove(self):
        if self.handle is not None:
            self.handle.remove()
            self.handle = None


def install_attention(pipe, config: PecoConfig):
    """Give every attention block of ``pipe.transformer`` a PecoAttention; return the shared context."""
    transformer = pipe.transformer
    old = getattr(transformer, _ATTRIBUTE, None)
    if old is not None:
        old.remove()
    attentions = [block.attn for block in (*transformer.transformer_blocks, *transformer.single_transformer_blocks)]
    context = InferenceContext()
    installation = _Installation(context, [PecoAttention(i, config, context) for i in range(len(attentions))],
                                 inspect.signature(transformer.forward))
    for attn, processor in zip(attentions, installation.processors):
        attn.set_processor(processor)
    installation.handle = transformer.register_forward_pre_hook(installation.before_forward, with_kwargs=True)
    setattr(transformer, _ATTRIBUTE, installation)
    return context


def reset_state(pipe):
    """Forget the step count and every layer's cached centroids (call before each new video)."""
    getattr(pipe.transformer, _ATTRIBUTE).reset()


_PROJECTIONS = ("to_q", "to_k", "to_v", "add_q_proj", "add_k_proj", "add_v_proj", "to_add_out")


def _projection_places(transformer):
    """(block's number, owner, name or index, layer) of every ``torch.nn.Linear`` among the blocks' projections."""
    places = {}
    for number, block in enumerate((*transformer.transformer_blocks, *transformer.single_transformer_blocks)):
        attn = block.attn
        out = getattr(attn, "to_out", None)
        own = [(attn, name, getattr(attn, name, None)) for name in (*_PROJECTIONS, "to_out")]
        if isinstance(out, (torch.nn.ModuleList, torch.nn.Sequential, list)) and len(out):
            own.append((out, 0, out[0]))
        for owner, key, layer in own:
            if type(layer) is torch.nn.Linear:
                places.setdefault((id(owner), key), (number, owner, key, layer))
    return list(places.values())


def _attached(layer):
    """Whether something hangs on this module that would be lost with it."""
    return "forward" in vars(layer) or any(
        (layer._forward_hooks, layer._forward_pre_hooks, layer._backward_hooks, layer._backward_pre_hooks))


def quantize_projections(pipe):
    """Put ``projection.Int8Linear`` in the place of every ``torch.nn.Linear`` among the projections of
    ``pipe.transformer``'s attention blocks (``to_out`` or its first layer too); return how many places. For inference.

    All layers are made before the first is replaced, so a layer that is refused (on the CPU, of more than 16384
    channels, with hooks or a ``forward`` of its own, which would be lost) leaves the transformer as it was. A layer in
    several places stays one.
    """
    places, made = _projection_places(pipe.transformer), {}
    for number, owner, key, layer in places:
        if _attached(layer):
            name = key if isinstance(key, str) else f"to_out.{key}"
            raise RuntimeError(f"attention of block {number}: {name} has hooks or a forward of its own, which an 8-bit "
                               "layer in its place would not have")
    for *_, layer in places:
        if id(layer) not in made:
            made[id(layer)] = projection.Int8Linear.from_linear(layer)
    for _, owner, key, layer in places:
        if isinstance(key, str):
            setattr(owner, key, made[id(layer)])
        else:
            owner[key] = made[id(layer)]
    return len(places)
