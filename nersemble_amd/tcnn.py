"""tcnn-shaped operator layer (``tinycudann`` Python API subset the reference imports):
``Network``, ``NetworkWithInputEncoding``, ``Encoding`` with ``.params`` (flat fp32 ``nn.Parameter``),
``.n_output_dims`` and fp16 outputs -- backed by the MFMA kernels of libnsx.so.

Reference call sites: nersemble_nerfacto_field.py:98-112 (direction encoding), :142-153 (mlp_base),
:162-172 (mlp_head).  Supported configurations are the ones the reference instantiates on the hot path:
FullyFusedMLP, 64 neurons, ReLU, 1-2 hidden layers, output None/Sigmoid, Identity encoding.
"""
import math

import torch
from torch import nn

from . import _lib, experts
from . import functional as F

_ACT = {"None": 0, "Sigmoid": 1}


def _xavier_flat(shapes, gen) -> torch.Tensor:
    parts = []
    for fan_out, fan_in in shapes:
        bound = math.sqrt(6.0 / (fan_in + fan_out))
        parts.append(((torch.rand(fan_out * fan_in, generator=gen) * 2 - 1) * bound))
    return torch.cat(parts)


class Network(nn.Module):
    """``tcnn.Network(n_input_dims, n_output_dims, network_config)`` (FullyFusedMLP)."""

    def __init__(self, n_input_dims: int, n_output_dims: int, network_config: dict, seed: int = 1337):
        super().__init__()
        if network_config.get("otype", "FullyFusedMLP") != "FullyFusedMLP":
            raise NotImplementedError("only FullyFusedMLP is provided")
        if network_config.get("n_neurons", 64) != 64 or network_config.get("activation", "ReLU") != "ReLU":
            raise NotImplementedError("native FullyFusedMLP: 64 neurons, ReLU (the reference's configuration)")
        n_hidden = int(network_config.get("n_hidden_layers", 1))
        if n_hidden not in (1, 2):
            raise NotImplementedError("native FullyFusedMLP supports 1 or 2 hidden layers")
        if n_input_dims > 32 or n_output_dims > 16:
            raise NotImplementedError("native FullyFusedMLP: n_input_dims <= 32, n_output_dims <= 16")
        self.n_input_dims, self.n_output_dims = n_input_dims, n_output_dims
        self.n_hidden_mats = n_hidden - 1
        self.out_act = _ACT[network_config.get("output_activation", "None")]
        gen = torch.Generator().manual_seed(seed)
        shapes = [(64, 32)] + [(64, 64)] * self.n_hidden_mats + [(16, 64)]
        self.params = nn.Parameter(_xavier_flat(shapes, gen))
        assert self.params.numel() == 64 * 32 + self.n_hidden_mats * 64 * 64 + 16 * 64

    def half_weights(self) -> torch.Tensor:
        """fp16 copy of ``params`` (what the kernels read), made once per optimizer step instead of once per call (tcnn
        itself casts its fp32 master parameters to fp16 on every step).  Fused optimizers update parameters without
        bumping ``Tensor._version``, hence the optimizer-step counter in the key."""
        from .field_components.deformation_field import _OPTIMIZER_STEPS
        p = self.params
        key = (p._version, p.data_ptr(), _OPTIMIZER_STEPS[0])
        if getattr(self, "_w16_key", None) != key:
            self._w16 = F.f32_to_f16(p.detach())
            self._w16_key = key
        return self._w16

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """x [B, n_input_dims] (fp16 or fp32) -> [B, n_output_dims] fp16."""
        x2 = x.reshape(-1, self.n_input_dims)
        if x2.dtype == torch.float16:
            return F.fused_mlp(self.params, self.n_hidden_mats, self.n_output_dims, self.out_act, b=x2)
        return F.fused_mlp(self.params, self.n_hidden_mats, self.n_output_dims, self.out_act, a=x2.float())


class NetworkWithInputEncoding(Network):
    """``tcnn.NetworkWithInputEncoding`` with the Identity encoding the reference uses for mlp_base when the
    HashEnsemble is enabled (nersemble_nerfacto_field.py:123-129)."""

    def __init__(self, n_input_dims: int, n_output_dims: int, encoding_config: dict, network_config: dict,
                 seed: int = 1337):
        if encoding_config.get("otype") != "Identity":
            raise NotImplementedError("native NetworkWithInputEncoding: Identity encoding (use HashEnsemble for grids)")
        super().__init__(n_input_dims, n_output_dims, network_config, seed)


class RoutedNetwork(nn.Module):
    """A sparse mixture of E fully connected networks of one shape, every row evaluated by ``top_k`` of them
    (``nersemble_amd.experts``) -- the routed counterpart of ``Network``, for widths that FullyFusedMLP does not have.

    ``network_config``: ``n_neurons`` (a multiple of 8), ``n_hidden_layers`` >= 1, ``activation`` ReLU, ``output_activation``
    None, ``otype`` CutlassMLP (tcnn's name for networks of any width).  ``routing_config``: ``n_experts``, ``top_k`` and,
    optionally, ``scores``, ``renormalise``, ``scale``, ``n_groups``, ``top_groups``, ``group_top`` (``route_experts``) and
    ``balance`` (off by default).

    ``params``: all experts' matrices, flat fp32, layer by layer [E][n_out][n_in] without biases, inputs and outputs padded to
    multiples of 8; ``gate`` [E, n_input_dims]: the router (logits = x gate^T in fp32); buffer ``balance`` [E], if asked for:
    added to the scores for the choice alone and moved by ``rebalance``."""

    def __init__(self, n_input_dims: int, n_output_dims: int, network_config: dict, routing_config: dict, seed: int = 1337):
        super().__init__()
        if network_config.get("otype", "CutlassMLP") != "CutlassMLP":
            raise NotImplementedError("RoutedNetwork: otype CutlassMLP (networks of any width)")
        if network_config.get("activation", "ReLU") != "ReLU" or network_config.get("output_activation", "None") != "None":
            raise NotImplementedError("RoutedNetwork: ReLU between the layers, no output activation")
        width, n_hidden = int(network_config.get("n_neurons", 64)), int(network_config.get("n_hidden_layers", 1))
        if width < 8 or width % 8 or n_hidden < 1 or n_input_dims < 1 or n_output_dims < 1:
            raise NotImplementedError("RoutedNetwork: n_neurons a multiple of 8, at least one hidden layer, input and output")
        cfg = dict(routing_config)
        self.n_experts, self.top_k = int(cfg.pop("n_experts")), int(cfg.pop("top_k"))
        if not 1 <= self.top_k <= min(self.n_experts, _lib.NSX_MAX_TOP_K) or self.n_experts > _lib.NSX_MAX_EXPERTS:
            raise NotImplementedError(f"RoutedNetwork: 1 <= top_k <= n_experts <= {_lib.NSX_MAX_EXPERTS}, top_k <= {_lib.NSX_MAX_TOP_K}")
        unknown = set(cfg) - {"scores", "renormalise", "scale", "n_groups", "top_groups", "group_top", "balance"}
        if unknown:
            raise NotImplementedError(f"RoutedNetwork: routing_config has no {sorted(unknown)}")
        balance = bool(cfg.pop("balance", False))
        self.routing = cfg
        self.n_input_dims, self.n_output_dims = n_input_dims, n_output_dims
        pad = lambda n: -(-n // 8) * 8                                       # noqa: E731
        dims = [pad(n_input_dims)] + [width] * n_hidden + [pad(n_output_dims)]
        self.shapes = [(self.n_experts, o, i) for i, o in zip(dims, dims[1:])]
        gen = torch.Generator().manual_seed(seed)
        self.params = nn.Parameter(_xavier_flat([(o, i) for e, o, i in self.shapes for _ in range(e)], gen))
        self.gate = nn.Parameter((torch.rand((self.n_experts, n_input_dims), generator=gen) * 2 - 1) / math.sqrt(n_input_dims))
        self.register_buffer("balance", torch.zeros(self.n_experts) if balance else None)
        self.register_buffer("load", torch.zeros(self.n_experts), persistent=False)

    def half_weights(self) -> torch.Tensor:
        """fp16 copy of ``params`` as they are now.  (Nothing is kept: the replays of a captured step change weights without a word.)"""
        return F.f32_to_f16(self.params.detach())

    def forward(self, x: torch.Tensor, selector: torch.Tensor = None) -> torch.Tensor:
        """x [B, n_input_dims] (fp16 or fp32) -> [B, n_output_dims] fp16; ``selector`` uint8 [B]: rows with 0 are not evaluated
        (their output is 0)."""
        x2 = x.reshape(-1, self.n_input_dims)
        if _lib.ndev_tensor(x2.shape[0]) is not None:
            raise RuntimeError("RoutedNetwork: the router's product runs over whole arrays, not over a device-side row count "
                               "(mask the rows behind it with `selector` instead)")
        if selector is not None:                    # (the gate's gradient is a product over all rows: 0 times what is not finite is not 0)
            x2 = torch.where(selector.reshape(-1, 1) != 0, x2, x2.new_zeros(()))
        with torch.autocast(device_type=x2.device.type, enabled=False):      # (a trainer's autocast would make the product in 16 bits)
            logits = x2.float() @ self.gate.t()
        weights, chosen = experts.route_experts(logits, self.top_k, bias=self.balance, selector=selector, **self.routing)
        plan = experts.expert_plan(chosen, self.n_experts)
        if self.training:
            self.load.copy_(plan.offsets[1:] - plan.offsets[:-1])
        h = x2.to(torch.float16)
        if self.shapes[0][2] != self.n_input_dims:
            h = nn.functional.pad(h, (0, self.shapes[0][2] - self.n_input_dims))
        sizes = [e * o * i for e, o, i in self.shapes]
        layers = zip(torch.split(self.params, sizes), torch.split(self.half_weights(), sizes), self.shapes)
        for n, (w, w16, shape) in enumerate(layers):
            h = experts.expert_linear(h, w.view(shape), plan, gather=n == 0, relu=n < len(sizes) - 1, w16=w16.view(shape))
        return experts.expert_combine(h, weights, plan)[:, :self.n_output_dims]

    @torch.no_grad()
    def rebalance(self, rate: float = 1e-3) -> None:
        """One step of the balancing bias against the load of the last training forward: experts above the mean load lose
        ``rate``, those below gain it."""
        if self.balance is None:
            raise RuntimeError("RoutedNetwork: routing_config has no balance")
        self.balance += rate * torch.sign(self.load.mean() - self.load)


class Encoding(nn.Module):
    """``tcnn.Encoding``: ``Identity`` (direction encoding with spherical_harmonics_degree = 0, the default of every
    shipped NeRSemble config, nersemble_instant_ngp.py:46), ``Frequency`` (the field's ``position_encoding``,
    nersemble_nerfacto_field.py:137-140 -- constructed by the reference, evaluated only under ``use_pred_normals``, which
    no NeRSemble config sets: constructed here too, never evaluated) and ``HashGrid`` with tcnn's parameter layout and
    U(-1e-4, 1e-4) initialisation (the operator the reference's own HashEnsemble instantiates at
    hash_ensemble.py:42-50; the fused ``nersemble_amd`` HashEnsemble is the fast path).

    Like every tcnn module, a parameter-free encoding registers an EMPTY flat ``params``: it is an entry of
    ``field.parameters()`` (hence of the ``fields`` optimizer group's numbering) and a key of the state dict
    (tests/golden/state_manifest.json, generated from the reference's module tree)."""

    def __init__(self, n_input_dims: int, encoding_config: dict, seed: int = 1337):
        super().__init__()
        otype = encoding_config.get("otype")
        self.otype = otype
        self.n_input_dims = n_input_dims
        if otype == "Identity":
            self.n_output_dims = n_input_dims
            self.params = nn.Parameter(torch.empty(0, dtype=torch.float32))
        elif otype == "Frequency":
            self.n_output_dims = n_input_dims * 2 * int(encoding_config["n_frequencies"])
            self.params = nn.Parameter(torch.empty(0, dtype=torch.float32))
        elif otype == "HashGrid":
            if n_input_dims != 3 or encoding_config.get("interpolation", "Linear") != "Linear":
                raise NotImplementedError("native HashGrid: 3-D input, Linear interpolation")
            self.f_enc = int(encoding_config.get("n_features_per_level", 2))
            if self.f_enc not in (2, 4, 8):
                raise NotImplementedError("native HashGrid: n_features_per_level in {2, 4, 8}")
            self.geom = _lib.grid_geometry(int(encoding_config.get("n_levels", 16)),
                                           float(encoding_config.get("per_level_scale", 2.0)),
                                           int(encoding_config.get("base_resolution", 16)),
                                           int(encoding_config.get("log2_hashmap_size", 19)))
            self.n_output_dims = self.geom.n_levels * self.f_enc
            gen = torch.Generator().manual_seed(seed)
            self.params = nn.Parameter((torch.rand(self.geom.total_entries * self.f_enc, generator=gen) * 2 - 1) * 1e-4)
        else:
            raise NotImplementedError(f"native Encoding: Identity, Frequency (construction only) and HashGrid (got {otype})")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.otype == "Identity":
            return x.to(torch.float16)
        if self.otype == "Frequency":
            raise NotImplementedError("tcnn Frequency encoding: only reached under use_pred_normals "
                                      "(nersemble_nerfacto_field.py:213-226), which NeRSemble never sets")
        return F.hashgrid_encoding(x, self.params.view(self.geom.total_entries, self.f_enc), self.f_enc, self.geom)
