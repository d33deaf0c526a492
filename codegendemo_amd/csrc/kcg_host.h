// kcg_host.h — what kcg_api.cc shares with the other host sources: the thread's error text and the HIP runtime it has bound.
#pragma once
#include <hip/hip_runtime_api.h>

#include <string>

namespace kcg {

struct HostHip {
  decltype(&::hipGetDevice) GetDevice;
  decltype(&::hipSetDevice) SetDevice;
  decltype(&::hipModuleLoadData) ModuleLoadData;
  decltype(&::hipModuleGetFunction) ModuleGetFunction;
  decltype(&::hipModuleUnload) ModuleUnload;
  decltype(&::hipModuleLaunchKernel) ModuleLaunchKernel;
  hipError_t (*FuncSetAttribute)(const void*, hipFuncAttribute, int);
};

// null, with the reason in the thread's error text, when no HIP runtime can be bound
const HostHip* host_hip();
int host_fail(int code, const std::string& msg);
int host_hip_fail(hipError_t e, const char* what);
void host_clear_error();

}  // namespace kcg
