"""MI355X (gfx950) implementation of CompactLogic's logic-layer hot path.

Same public modules as the reference package `compactlogic` (compactlogic/__init__.py:1):
LogicLayer, ConvLayer, GroupSum and the autograd bridges LogicLayerCudaFunction and
ConvLayerCudaFunction, plus the packed-bit inference API (PackBitsTensor), and the logic-tree
conv blocks of the third-party ConvLogic package (ConvLogicLayer, TreeLogicLayer,
PoolLogicLayer).  Beside the reference's modules: losses for training by reward or preference
(policy.py), dropout between logic layers (dropout_layer.py), recurrences over sequences
(recurrence.py), the verification of drafted actions (drafts.py), fused optimizer steps (optim.py).
All numerics run in libcompactlogic_hip.so, built in-tree (with the C++ side of the calls of all of
these but FusedAdam, csrc/autograd.cpp) by ``python -m compactlogic_amd.build``.
"""
from . import checkpoint, circuit, convlogic_hip, difflogic_hip
from .dropout_layer import Dropout, dropout
from .drafts import verify_drafts
from .layers import (ConvLayer, ConvLayerCudaFunction, ConvLayerSoftmaxFunction,
                     ConvLayerWindowFunction, GroupSum, GroupSumCrossEntropyFunction,
                     GroupSumFunction, LogicGroupSumCrossEntropyFunction, LogicLayer,
                     LogicLayerCudaFunction, LogicLayerRunsFunction, PackBitsTensor,
                     logic_group_sum_cross_entropy, sequential_cross_entropy)
from .optim import FusedAdam, FusedAdamW
from .packed_net import PackedNetwork
from .plan import RunPlan, build_run_plan
from .policy import policy_loss, preference_loss, selected_log_probs
from .recurrence import LogicRecurrence, gated_recurrence
from .schedules import (EntropyRowResampler, FixedSequentialEntropyFreezer,
                        SequentialEntropyFreezer)
from .treelogic import (ConvLogicFunction, ConvLogicLayer, FullConvLogicFunction,
                        PoolLogicLayer, TreeLogicFunction, TreeLogicLayer)

__all__ = [
    "LogicLayer", "GroupSum", "LogicLayerCudaFunction", "LogicLayerRunsFunction",
    "GroupSumCrossEntropyFunction", "GroupSumFunction", "PackBitsTensor", "RunPlan", "build_run_plan", "difflogic_hip",
    "ConvLayer", "ConvLayerCudaFunction", "ConvLayerSoftmaxFunction", "ConvLayerWindowFunction",
    "convlogic_hip", "SequentialEntropyFreezer", "FixedSequentialEntropyFreezer",
    "EntropyRowResampler", "PackedNetwork", "ConvLogicLayer", "TreeLogicLayer", "PoolLogicLayer",
    "ConvLogicFunction", "FullConvLogicFunction", "TreeLogicFunction", "FusedAdam", "FusedAdamW",
    "LogicGroupSumCrossEntropyFunction", "logic_group_sum_cross_entropy",
    "sequential_cross_entropy", "checkpoint", "circuit", "Dropout", "dropout",
    "policy_loss", "preference_loss", "selected_log_probs",
    "LogicRecurrence", "gated_recurrence", "verify_drafts",
]
