// kq_host.h -- host-side services of kq_api.cu that the library's other translation units share.
#pragma once
#include <string>

// Sets this thread's kq_error() text and returns `code`.
int kqh_error(int code, const std::string& msg);

struct KqhDevice {
  int nsm;             // multiprocessors
  int* err;            // two words: the serving operators' error word on this device (KQ_DEV_ERR_* bits), and a place to
};                     // take it to
// Initialises `device` on first use, makes it current and describes it; a KQ_* status.
int kqh_device(int device, KqhDevice* out);

// What the operators' kernels flagged, in words (the bits of device operands alone).
std::string kqh_operands(int bits);

// A model's operators leave their flags in its own error word (`err`), which its own steps read: the flags of
// other callers on the device stay theirs.
struct kq_pages;
// kq_pages_create with another handle's attention scratch (null: its own): the handles' calls share a stream.
kq_pages* kqh_pages_create(const void* desc, int device, const kq_pages* with, int* err);
// kq_logit_rules (a kq_rule_args); its checks of the arguments alone.
int kqh_rules_check(const void* args);
int kqh_logit_rules(const void* args, int device, int* err, void* stream);
