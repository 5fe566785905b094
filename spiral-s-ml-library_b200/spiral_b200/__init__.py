"""spiral_b200: B200 (sm_100a) dense-matmul / policy-MLP path behind the reference's call surface.

A thin ctypes host over libspiral_b200.so (hand-written CUDA: tcgen05 MMAs with
TMEM accumulators fed by TMA).  No CPU fallback exists: without the built
library every operation raises.
"""
from ._lib import SpiralError, LIB_PATH  # noqa: F401
from .device import (DeviceArray, Event, Stream, wait_event, GemmProfile, launch_count, device_count, device_ptr, device_status, check_device, mem_info, set_device, sm_count,  # noqa: F401
                     synchronize)
from .matmul import (dequantize_int4, gated, gated_grad, gated_grad_plan, gated_grad_workspace, gated_plan, head_spec, matmul, matmul_fp8, matmul_fp8_plan,  # noqa: F401
                     matmul_head, matmul_int4, matmul_int4_plan, matmul_plan, matmul_tf32, quantize_fp8, quantize_int4)
from . import primitives  # noqa: F401
from .models import EnsemblePolicyMLP, PolicyMLP, TokenPolicy, param_offsets, to_storage  # noqa: F401
from . import layers  # noqa: F401
from .optim import AdamW  # noqa: F401
from .parallel import DataParallel, PeerUpdate, shard_rows, bucket_ranges, update_slice  # noqa: F401
