from .functional import adamw, clip_grad_norm_, clip_grads, clip_grads_with_norm_, get_total_norm
from .muon_adamw import (MuonAdamW, MuonShardPlan, is_default_muon_parameter, mark_muon_parameters,
                         zeropower_via_newtonschulz5)

__all__ = ["MuonAdamW", "mark_muon_parameters", "MuonShardPlan", "is_default_muon_parameter",
           "zeropower_via_newtonschulz5", "adamw", "clip_grad_norm_", "clip_grads", "clip_grads_with_norm_",
           "get_total_norm"]
