"""graphgps_amd -- the GPSLayer hot path of rampasek/GraphGPS, built MI355X-first.

Importing the package registers the HIP-backed implementations under the reference's own
GraphGym plugin names (``network_dict['GPSModel']``, ``layer_dict['gatedgcnconv']``,
``layer_dict['gineconv']``, heads, encoders, losses).  Scope and boundary: DESIGN.md.
"""
__version__ = "0.1.0"

from .graphgym import register  # noqa: F401
from .graphgym.config import cfg, load_cfg, set_cfg  # noqa: F401
from .data import Batch  # noqa: F401
from .layer.gps_layer import GPSLayer  # noqa: F401
from .layer.gatedgcn_layer import GatedGCNLayer, GatedGCNGraphGymLayer  # noqa: F401
from .layer.gine_conv_layer import GINEConv, GINEConvLayer, GINEConvGraphGymLayer  # noqa: F401
from .network.gps_model import GPSModel  # noqa: F401
from .network.custom_gnn import CustomGNN  # noqa: F401
from .encoder import graphormer_encoder as _graphormer_encoder  # noqa: F401
from .encoder import extra_encoders as _extra_encoders  # noqa: F401
from .encoder import signnet_encoder as _signnet_encoder  # noqa: F401
from .head import edge_head as _edge_head, heads as _heads  # noqa: F401
from .layer.graphormer_layer import GraphormerLayer  # noqa: F401
from .network.graphormer import GraphormerModel  # noqa: F401
from .network.san_transformer import SANTransformer  # noqa: F401
from .loss import losses as _losses  # noqa: F401
from .optim import FlatAdamW, FlatAdamW8bit, ParamArena  # noqa: F401
from . import schedulers as _schedulers  # noqa: F401

import os as _os

CONFIG_DIR = _os.path.join(_os.path.dirname(_os.path.abspath(__file__)), "configs")


def create_model(cfg_file=None, opts=None, dim_in=None, dim_out=None):
    """``set_cfg`` + ``load_cfg`` + ``network_dict[cfg.model.type](dim_in, dim_out)``: the
    GraphGym ``create_model`` path (reference main.py:118-121,144) without the dataset."""
    set_cfg(cfg)
    load_cfg(cfg, cfg_file, opts)
    if dim_in is not None:
        cfg.share.dim_in = dim_in
    if dim_out is not None:
        cfg.share.dim_out = dim_out
    return register.network_dict[cfg.model.type](cfg.share.dim_in, cfg.share.dim_out)


def enable_gemm_tuning(filename=None, max_ms_per_solution=30):
    """Let PyTorch's TunableOp time the rocBLAS / hipBLASLt solutions for every dense-projection
    GEMM shape of the block at its first call and dispatch to the fastest from then on (results
    cached in ``filename``).  The libraries' default heuristics leave 20-40 % on the table at the
    PCQM4M shapes ([7569 x 384] x [384 x 2688]: 157 -> 125 us; out_proj [7569 x 384 x 384]:
    44 -> 25 us on MI355X).  Call once before the first training step; call
    ``torch.cuda.tunable.tuning_enable(False)`` after the warm-up steps to freeze the choice."""
    import tempfile
    import torch
    t = torch.cuda.tunable
    t.enable(True)
    t.tuning_enable(True)
    t.set_max_tuning_duration(int(max_ms_per_solution))
    # one results file per process: ranks of a data-parallel job tune (and write) independently
    rank = _os.environ.get("LOCAL_RANK", _os.environ.get("RANK", "0"))
    t.set_filename(filename or _os.path.join(tempfile.gettempdir(), f"graphgps_amd_tunableop_r{rank}.csv"))
    return t
