from .base_ranking_model import BaseRankingModel, ActivationFunctions, NormalizationFunctions, Initializer
from .DNN import DNN
from .Linear import Linear
from .normalization import layer_norm, layer_norm_backward, layer_norm_workspace
