from .attention_packed import attention_packed
from .continuous_count import continuous_count
from .rmsnorm import fused_residual_add_rmsnorm, rmsnorm
from .sequence_packing import pack_sequence, unpack_sequence
from .swiglu import swiglu
from .swiglu_packed import swiglu_packed
