// Launch attributes, and the device side of launches that overlap.
#pragma once
#include <cuda_runtime.h>

namespace psb {

namespace {

// Programmatic dependent launch: a kernel that was allowed to start beside its predecessor's tail (`start_early`) touches no global
// memory before wait_predecessor() has returned. It allows its own successor to start once its TMEM is allocated in every CTA: a
// successor that got the TMEM first would wait for this kernel, and this kernel for the TMEM.
__device__ __forceinline__ void wait_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void allow_successor() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

inline cudaLaunchAttribute start_early() {
    cudaLaunchAttribute a = {};
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
    return a;
}
inline cudaLaunchAttribute in_clusters(int size) {
    cudaLaunchAttribute a = {};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = size;
    a.val.clusterDim.y = 1;
    a.val.clusterDim.z = 1;
    return a;
}

}  // namespace

}  // namespace psb
