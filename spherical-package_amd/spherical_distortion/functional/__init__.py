from .mapped_ops import (mapped_convolution, mapped_transposed_convolution,  # noqa: F401
                         mapped_max_pool, mapped_max_unpool, mapped_avg_pool,
                         mapped_avg_unpool, resample, unresample, uv_resample, voting_resample, MappedConvolutionFunction,
                         MappedTransposedConvolutionFunction, MappedMaxPoolFunction,
                         MappedMaxUnpoolFunction,
                         MappedAvgPoolFunction, MappedAvgUnpoolFunction, ResampleFunction,
                         UnresampleFunction, UVResampleFunction)
from .token_ops import (bucket_attention, add_rms_norm, add_rms_norm_quantized, dequantize_rows,  # noqa: F401
                        adamw_step, adamw_step_8bit, adamw_moment_values, BucketAttentionFunction,
                        AddRMSNormFunction)
