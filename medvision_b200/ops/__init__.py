from .roi_align_nd import RoIAlign
from .roi_align_rotated_nd import RoIAlignRotated
from .cuda_fun_tools import (affine_2d, affine_3d, affine_fields_3d, affine_label_2d, affine_label_3d,
                             apply_offset_2d, apply_offset_3d)
from .host_pipeline import affine_from_host
from .cross_attention import cross_attention
from .dropout import Dropout, dropout
from .group_norm import GroupNorm, group_norm
from .label_log_probs import LabelLogProbs, label_log_probs
from .rotary_positions import rotary_positions
from .window_attention import window_attention

__all__ = ['RoIAlign', 'RoIAlignRotated', 'affine_2d', 'affine_3d', 'affine_from_host', 'apply_offset_2d', 'apply_offset_3d', 'affine_label_2d',
           'affine_label_3d', 'affine_fields_3d', 'cross_attention', 'Dropout', 'dropout', 'GroupNorm', 'group_norm', 'LabelLogProbs',
           'label_log_probs', 'rotary_positions', 'window_attention']
