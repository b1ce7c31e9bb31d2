"""MLP target (hyper/target/mlp.py:7-29): a SequentialModule of batched Linear layers."""
from ..layers.linear import FinalLinear, Linear
from ..layers.module import SequentialModule, register_gen_module
from ..layers.norm import LayerNorm


@register_gen_module('mlp')
class MLPModule(SequentialModule):
    """norm / compute / checkpoint (not in the reference's signature; each also per layer): norm='layer_norm' puts a LayerNorm in front
    of a layer (given for the whole MLP: of every layer but the first), compute and checkpoint are Linear's."""

    def __init__(self, layers, activation='relu', act_last=False, track=True, norm=None, compute='fp32', checkpoint=None):
        last = len(layers) - 1
        modules = []
        for i, layer in enumerate(layers):
            layer_norm = layer.get('norm', norm if i > 0 else None)
            if layer_norm not in (None, 'layer_norm'):
                raise ValueError("norm is None or 'layer_norm', got %r" % (layer_norm,))
            if layer_norm is not None:
                modules.append(LayerNorm(layer['in'], track=False))
            modules.append((FinalLinear if layer.get('last', False) else Linear)(
                in_features=layer['in'], out_features=layer['out'], bias=layer.get('bias', True),
                act=layer.get('act', None if (i == last and not act_last) else activation),
                gamma=layer.get('gamma', None if i == 0 else activation), track=layer.get('track', True),
                compute=layer.get('compute', compute), checkpoint=layer.get('checkpoint', checkpoint)))
        super().__init__(modules=modules, track=track)

    @staticmethod
    def from_config(config):
        return config
