"""minitensor_b200 -- B200 (sm_100a) engine for miniTensor's fp32 GEMM path.

The kernels and the C ABI live in ``csrc/`` (built into ``libmtgemm.so``; the ABI is
declared in ``include/mtgemm.h``). ``engine`` mirrors the reference's GPU entry points on
top of it, ``lowbit`` has the 8-bit and 4-bit forms of Linear and the RMS norm before it,
``sharded`` splits large GEMMs over several GPUs, ``inputs`` makes the seeded synthetic
workloads.
"""
from . import engine  # noqa: F401
from .engine import (  # noqa: F401
    bmm, bmm_gpu, gemm, linear_backward, linear_forward, linear_fwd_gpu, matmul, matmul_gpu,
    matmul_gpu_bk16, matmul_gpu_strided, matmul_gpu_v2,
)
from .lowbit import (  # noqa: F401
    Q4Weight, Q8Tensor, RmsNorm, dequantize_q4, dequantize_q8, linear_backward_q8, linear_forward_q4,
    linear_forward_q8, linear_weight_grad_q8, quantize_q4, quantize_q8, rms_norm, rms_norm_backward,
)
