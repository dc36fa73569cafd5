"""Host mirror of ``monoloco.train`` for the training step (reference monoloco/train/__init__.py)."""
from .adamw import AdamW, adamw_step, state_scales
from .hip_trainer import HipTrainer
from .trainer import KeypointsDataset, Trainer

__all__ = ['AdamW', 'HipTrainer', 'Trainer', 'KeypointsDataset', 'adamw_step', 'state_scales']
