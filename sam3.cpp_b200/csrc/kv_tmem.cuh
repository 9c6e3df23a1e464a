// TMEM loads and stores, and the lane that issues, of the tensor-core kernels over the quantised key / value cache.
#pragma once
#include "kv_attention.cuh"

namespace s3b {

#define KV_TMEM_LD32(taddr, R)                                                                               \
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "                                                     \
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"                                     \
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"                    \
               : "=r"((R)[0]), "=r"((R)[1]), "=r"((R)[2]), "=r"((R)[3]), "=r"((R)[4]), "=r"((R)[5]),         \
                 "=r"((R)[6]), "=r"((R)[7]), "=r"((R)[8]), "=r"((R)[9]), "=r"((R)[10]), "=r"((R)[11]),       \
                 "=r"((R)[12]), "=r"((R)[13]), "=r"((R)[14]), "=r"((R)[15]), "=r"((R)[16]), "=r"((R)[17]),   \
                 "=r"((R)[18]), "=r"((R)[19]), "=r"((R)[20]), "=r"((R)[21]), "=r"((R)[22]), "=r"((R)[23]),   \
                 "=r"((R)[24]), "=r"((R)[25]), "=r"((R)[26]), "=r"((R)[27]), "=r"((R)[28]), "=r"((R)[29]),   \
                 "=r"((R)[30]), "=r"((R)[31])                                                                \
               : "r"(taddr))
#define KV_TMEM_ST32(taddr, R)                                                                               \
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "                                               \
               "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"                                    \
               "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),             \
               "r"((R)[0]), "r"((R)[1]), "r"((R)[2]), "r"((R)[3]), "r"((R)[4]), "r"((R)[5]), "r"((R)[6]),    \
               "r"((R)[7]), "r"((R)[8]), "r"((R)[9]), "r"((R)[10]), "r"((R)[11]), "r"((R)[12]),              \
               "r"((R)[13]), "r"((R)[14]), "r"((R)[15]), "r"((R)[16]), "r"((R)[17]), "r"((R)[18]),           \
               "r"((R)[19]), "r"((R)[20]), "r"((R)[21]), "r"((R)[22]), "r"((R)[23]), "r"((R)[24]),           \
               "r"((R)[25]), "r"((R)[26]), "r"((R)[27]), "r"((R)[28]), "r"((R)[29]), "r"((R)[30]),           \
               "r"((R)[31])                                                                                  \
               : "memory")
#define KV_TMEM_ST8(taddr, R)                                                                                \
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),        \
               "r"((R)[0]), "r"((R)[1]), "r"((R)[2]), "r"((R)[3]), "r"((R)[4]), "r"((R)[5]), "r"((R)[6]),    \
               "r"((R)[7])                                                                                   \
               : "memory")
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
#define KV_TMEM_ST16(taddr, R)                                                                               \
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "                                               \
               "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),                     \
               "r"((R)[0]), "r"((R)[1]), "r"((R)[2]), "r"((R)[3]), "r"((R)[4]), "r"((R)[5]), "r"((R)[6]),    \
               "r"((R)[7]), "r"((R)[8]), "r"((R)[9]), "r"((R)[10]), "r"((R)[11]), "r"((R)[12]),              \
               "r"((R)[13]), "r"((R)[14]), "r"((R)[15])                                                      \
               : "memory")
// One lane of a converged warp, always the same. The compiler then knows that a single lane runs what follows and feeds the
// MMAs from uniform registers: 78 clocks for a 128 x 128 x 16 product from TMEM, against 168 behind `lane == 0`.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

}  // namespace s3b
