// Single translation unit of libspiral_b200.so: the kernels share one device
// status word and a few launch helpers, so they are compiled together without
// relocatable device code.
#include "runtime.cu"
#include "rowops.cu"
#include "gemm_fp32.cu"
#include "gemm_umma.cu"
#include "api.cu"
#include "mlp.cu"
#include "mlp_fused.cu"
#include "dp.cu"
#include "embedding.cu"
#include "layer_norm.cu"
#include "adamw.cu"
#include "gemm_fp8.cu"
#include "log_probs.cu"
#include "gated.cu"
#include "gemm_int4.cu"
#include "selftest.cu"
