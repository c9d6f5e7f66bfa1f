// Stand-in for the C interface of XLA's FFI, for builds without an XLA checkout.
//
// It declares the structs, numbers and function-table entries that ffi_handlers.cc and mock_ffi_runtime.cc use, and
// nothing else, so that the handlers can be built and driven by the mock runtime where XLA's own headers are not at
// hand.  Both libraries of such a build agree with each other; the order of the fields is this file's own.  A process
// that holds the real XLA needs a build against its headers (`make XLA_ROOT=<xla checkout>`).  A mixed pair is refused: the
// version number below is one that no XLA has, and b200sd_ffi_register compares it; and a call frame's size, which is the
// first field of everybody's frames, has a mark above any real size, without which a handler leaves a frame alone.
#ifndef B200SD_FFI_STANDIN_C_API_H_
#define B200SD_FFI_STANDIN_C_API_H_

#include <stddef.h>
#include <stdint.h>

#define B200SD_FFI_STANDIN 1
#define XLA_FFI_API_MAJOR 0x7b20
#define XLA_FFI_API_MINOR 1

extern "C" {

struct XLA_FFI_Api;
struct XLA_FFI_Error;           // defined by the runtime
struct XLA_FFI_InvokeContext;   // defined by the runtime

// absl::StatusCode numbers.
enum XLA_FFI_Error_Code {
  XLA_FFI_Error_Code_OK = 0,
  XLA_FFI_Error_Code_UNKNOWN = 2,
  XLA_FFI_Error_Code_INVALID_ARGUMENT = 3,
  XLA_FFI_Error_Code_NOT_FOUND = 5,
  XLA_FFI_Error_Code_ALREADY_EXISTS = 6,
  XLA_FFI_Error_Code_FAILED_PRECONDITION = 9,
  XLA_FFI_Error_Code_UNIMPLEMENTED = 12,
  XLA_FFI_Error_Code_INTERNAL = 13,
};

// xla::PrimitiveType numbers.
enum XLA_FFI_DataType {
  XLA_FFI_DataType_INVALID = 0,
  XLA_FFI_DataType_PRED = 1,
  XLA_FFI_DataType_S8 = 2,
  XLA_FFI_DataType_S32 = 4,
  XLA_FFI_DataType_S64 = 5,
  XLA_FFI_DataType_U8 = 6,
  XLA_FFI_DataType_F16 = 10,
  XLA_FFI_DataType_F32 = 11,
  XLA_FFI_DataType_F64 = 12,
  XLA_FFI_DataType_BF16 = 16,
  XLA_FFI_DataType_F8E5M2 = 19,
  XLA_FFI_DataType_F8E4M3FN = 20,
  XLA_FFI_DataType_F8E8M0FNU = 33,
};

enum XLA_FFI_AttrType { XLA_FFI_AttrType_ARRAY = 1, XLA_FFI_AttrType_SCALAR = 3, XLA_FFI_AttrType_STRING = 4 };
enum XLA_FFI_ArgType { XLA_FFI_ArgType_BUFFER = 1 };
enum XLA_FFI_RetType { XLA_FFI_RetType_BUFFER = 1 };
enum XLA_FFI_ExecutionStage {
  XLA_FFI_ExecutionStage_INSTANTIATE = 0,
  XLA_FFI_ExecutionStage_PREPARE = 1,
  XLA_FFI_ExecutionStage_INITIALIZE = 2,
  XLA_FFI_ExecutionStage_EXECUTE = 3,
};

struct XLA_FFI_ByteSpan { const char* ptr; size_t len; };
struct XLA_FFI_Scalar { XLA_FFI_DataType dtype; void* value; };
struct XLA_FFI_Array { XLA_FFI_DataType dtype; size_t size; void* data; };

struct XLA_FFI_Buffer {
  size_t struct_size;
  XLA_FFI_DataType dtype;
  void* data;
  int64_t rank;
  int64_t* dims;
};

// ---- the call frame --------------------------------------------------------------------------
enum XLA_FFI_Extension_Type { XLA_FFI_Extension_Metadata = 1 };
struct XLA_FFI_Extension_Base {
  size_t struct_size;
  XLA_FFI_Extension_Type type;
  XLA_FFI_Extension_Base* next;
};
struct XLA_FFI_Api_Version { size_t struct_size; int major_version, minor_version; };

typedef uint32_t XLA_FFI_Handler_Traits;
enum { XLA_FFI_HANDLER_TRAITS_COMMAND_BUFFER_COMPATIBLE = 1 };
struct XLA_FFI_Metadata {
  size_t struct_size;
  XLA_FFI_Api_Version api_version;
  XLA_FFI_Handler_Traits traits;
};
struct XLA_FFI_Metadata_Extension {
  XLA_FFI_Extension_Base extension_base;
  XLA_FFI_Metadata* metadata;
};

struct XLA_FFI_Args { size_t struct_size; int64_t size; XLA_FFI_ArgType* types; void** args; };
struct XLA_FFI_Rets { size_t struct_size; int64_t size; XLA_FFI_RetType* types; void** rets; };
struct XLA_FFI_Attrs {
  size_t struct_size;
  int64_t size;
  XLA_FFI_AttrType* types;
  XLA_FFI_ByteSpan** names;
  void** attrs;
};
struct XLA_FFI_CallFrame {
  size_t struct_size;
  XLA_FFI_Extension_Base* extension_start;
  const XLA_FFI_Api* api;
  XLA_FFI_InvokeContext* ctx;
  XLA_FFI_ExecutionStage stage;
  XLA_FFI_Args args;
  XLA_FFI_Rets rets;
  XLA_FFI_Attrs attrs;
};

typedef XLA_FFI_Error* XLA_FFI_Handler(XLA_FFI_CallFrame*);
struct XLA_FFI_Handler_Bundle {
  XLA_FFI_Handler *instantiate, *prepare, *initialize, *execute;
};

// ---- the function table ----------------------------------------------------------------------
struct XLA_FFI_Error_Create_Args { size_t struct_size; const char* message; XLA_FFI_Error_Code errc; };
struct XLA_FFI_Error_GetDetails_Args { size_t struct_size; XLA_FFI_Error* error; const char* message; XLA_FFI_Error_Code errc; };
struct XLA_FFI_Error_Destroy_Args { size_t struct_size; XLA_FFI_Error* error; };
struct XLA_FFI_Handler_Register_Args {
  size_t struct_size;
  XLA_FFI_ByteSpan name, platform;
  XLA_FFI_Handler_Bundle bundle;
  XLA_FFI_Handler_Traits traits;
};
struct XLA_FFI_Stream_Get_Args { size_t struct_size; XLA_FFI_InvokeContext* ctx; void* stream; };
struct XLA_FFI_DeviceOrdinal_Get_Args { size_t struct_size; XLA_FFI_InvokeContext* ctx; int32_t device_ordinal; };
struct XLA_FFI_RunId_Get_Args { size_t struct_size; XLA_FFI_InvokeContext* ctx; int64_t run_id; };
struct XLA_FFI_TypeId { int64_t type_id; };
struct XLA_FFI_Type_Register_Args { size_t struct_size; XLA_FFI_TypeId* type_id; };
struct XLA_FFI_State_Set_Args { size_t struct_size; XLA_FFI_InvokeContext* ctx; XLA_FFI_ExecutionStage stage; XLA_FFI_TypeId* type_id; void* state; };
struct XLA_FFI_State_Get_Args { size_t struct_size; XLA_FFI_InvokeContext* ctx; XLA_FFI_ExecutionStage stage; XLA_FFI_TypeId* type_id; void* state; };
struct XLA_FFI_InvokeContext_FindExtension_Args { size_t struct_size; XLA_FFI_InvokeContext* ctx; void* extension; };
struct XLA_FFI_InvokeContext_Get_Args;
struct XLA_FFI_DeviceMemory_Allocate_Args;
struct XLA_FFI_DeviceMemory_Free_Args;
struct XLA_FFI_ThreadPool_Schedule_Args;
struct XLA_FFI_ThreadPool_NumThreads_Args;
struct XLA_FFI_Future_Create_Args;
struct XLA_FFI_Future_SetAvailable_Args;
struct XLA_FFI_Future_SetError_Args;

#define B200SD_FFI_ENTRY(name) XLA_FFI_Error* (*XLA_FFI_##name)(XLA_FFI_##name##_Args*)
struct XLA_FFI_Api {
  size_t struct_size;
  XLA_FFI_Api_Version api_version;
  B200SD_FFI_ENTRY(Error_Create);
  void (*XLA_FFI_Error_GetDetails)(XLA_FFI_Error_GetDetails_Args*);
  void (*XLA_FFI_Error_Destroy)(XLA_FFI_Error_Destroy_Args*);
  B200SD_FFI_ENTRY(Handler_Register);
  B200SD_FFI_ENTRY(Stream_Get);
  B200SD_FFI_ENTRY(Type_Register);
  B200SD_FFI_ENTRY(InvokeContext_Get);
  B200SD_FFI_ENTRY(State_Set);
  B200SD_FFI_ENTRY(State_Get);
  B200SD_FFI_ENTRY(DeviceMemory_Allocate);
  B200SD_FFI_ENTRY(DeviceMemory_Free);
  B200SD_FFI_ENTRY(ThreadPool_Schedule);
  B200SD_FFI_ENTRY(ThreadPool_NumThreads);
  B200SD_FFI_ENTRY(Future_Create);
  B200SD_FFI_ENTRY(Future_SetAvailable);
  B200SD_FFI_ENTRY(Future_SetError);
  B200SD_FFI_ENTRY(RunId_Get);
  B200SD_FFI_ENTRY(DeviceOrdinal_Get);
  B200SD_FFI_ENTRY(InvokeContext_FindExtension);
};
#undef B200SD_FFI_ENTRY

}  // extern "C"

#define XLA_FFI_Api_STRUCT_SIZE sizeof(XLA_FFI_Api)
#define XLA_FFI_Api_Version_STRUCT_SIZE sizeof(XLA_FFI_Api_Version)
#define XLA_FFI_Args_STRUCT_SIZE sizeof(XLA_FFI_Args)
#define XLA_FFI_Attrs_STRUCT_SIZE sizeof(XLA_FFI_Attrs)
#define XLA_FFI_Buffer_STRUCT_SIZE sizeof(XLA_FFI_Buffer)
#define XLA_FFI_CallFrame_STRUCT_SIZE (sizeof(XLA_FFI_CallFrame) | size_t{XLA_FFI_API_MAJOR} << 32)
#define XLA_FFI_Error_Destroy_Args_STRUCT_SIZE sizeof(XLA_FFI_Error_Destroy_Args)
#define XLA_FFI_Error_GetDetails_Args_STRUCT_SIZE sizeof(XLA_FFI_Error_GetDetails_Args)
#define XLA_FFI_Metadata_STRUCT_SIZE sizeof(XLA_FFI_Metadata)
#define XLA_FFI_Metadata_Extension_STRUCT_SIZE sizeof(XLA_FFI_Metadata_Extension)
#define XLA_FFI_Rets_STRUCT_SIZE sizeof(XLA_FFI_Rets)

#endif  // B200SD_FFI_STANDIN_C_API_H_
