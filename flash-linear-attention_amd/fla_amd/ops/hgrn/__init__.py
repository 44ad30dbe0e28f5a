from .chunk import chunk_hgrn
from .fused_recurrent import fused_recurrent_hgrn

__all__ = ['chunk_hgrn', 'fused_recurrent_hgrn']
