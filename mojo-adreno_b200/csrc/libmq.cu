// libmq.so is one translation unit: the kernels share the device status word (g_status) without
// relocatable device code, and each file keeps its helpers in its own namespace.
#include <algorithm>

#include "capi.cu"
#include "unpack.cu"
#include "gemv_q4.cu"
#include "tgemv.cu"
#include "gemm_q4.cu"
#include "moe.cu"
#include "pack.cu"
#include "io.cu"
#include "ep.cu"
#include "gemm_w8a8.cu"
#include "norm.cu"
#include "beam.cu"
#include "kv.cu"
#include "attn.cu"
#include "attn_tile.cu"
#include "verify.cu"
