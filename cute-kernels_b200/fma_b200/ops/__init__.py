from .continuous_count import continuous_count
from .fp8 import grouped_linear_fp8, linear_fp8, quantize_fp8, quantize_fp8_weight, swiglu_fp8_checkpoint
from .grouped_gemm import grouped_gemm
from .swiglu import swiglu, swiglu_packed
from .sequence_packing import pack_sequence, unpack_sequence
