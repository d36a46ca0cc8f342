// kq_host.h -- host-side services of kq_api.cu that the library's other translation units share.
#pragma once
#include <string>

// Sets this thread's kq_error() text and returns `code`.
int kqh_error(int code, const std::string& msg);

struct KqhDevice {
  int nsm;             // multiprocessors
  int* err;            // the serving operators' error word on this device (KQ_DEV_ERR_* bits)
};
// Initialises `device` on first use, makes it current and describes it; a KQ_* status.
int kqh_device(int device, KqhDevice* out);

struct kq_pages;
// kq_pages_create with another handle's attention scratch (null: its own): the handles' calls share a stream,
// and `with` is freed last.
kq_pages* kqh_pages_create(const void* desc, int device, const kq_pages* with);
