/*
 * check_program.c -- a resident program's control blocks on a machine without a GPU.  The device calls that the
 * library's resident program makes are defined here, over host memory, and take the place of the library's own;
 * tests/test_training_edges.py builds this with gcc and looks at what it prints.
 *
 *   check_program GRAPH.json KEEP,KEEP,...
 *
 * Prints the control block each planned call gets ("call NAME OFFSET", -1 for none), sets every word of the control
 * blocks, and prints tc_program_check's status, how many words it left set, and the status of a second check.
 */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "tcb200.h"

struct tc_buf { void* p; uint64_t bytes; };
static struct { uint64_t p, bytes; } last_clear;
static char names[4096][64];
static uint64_t ctrl[4096];
static int calls;

int tc_alloc(tc_ctx* ctx, uint64_t bytes, uint64_t canary, tc_buf** out) {
  tc_buf* b = (tc_buf*)malloc(sizeof *b);
  b->p = aligned_alloc(256, (bytes + canary + 255) / 256 * 256);
  b->bytes = bytes;
  *out = b;
  return 0;
}
int tc_buf_ptr(tc_buf* b, uint64_t* out) { *out = (uint64_t)b->p; return 0; }
int tc_free(tc_buf* b) { free(b->p); free(b); return 0; }
int tc_memset32(tc_ctx* ctx, uint64_t dst, uint32_t value, uint64_t count) {
  for (uint64_t i = 0; i < count; ++i) ((uint32_t*)dst)[i] = value;
  last_clear.p = dst;
  last_clear.bytes = 4 * count;
  return 0;
}
int tc_memcpy_htod(tc_ctx* ctx, uint64_t dst, const void* src, uint64_t bytes) { memcpy((void*)dst, src, bytes); return 0; }
int tc_memcpy_dtoh(tc_ctx* ctx, void* dst, uint64_t src, uint64_t bytes) { memcpy(dst, (void*)src, bytes); return 0; }
int tc_sync(tc_ctx* ctx, int timeout_ms) { return 0; }
int tc_compile_cubin(const char* src, void* out, uint64_t cap, uint64_t* n, char* log, size_t log_cap) {
  *n = 1;
  if (out) *(char*)out = 0;
  return 0;
}
int tc_module_load(tc_ctx* ctx, const void* cubin, uint64_t bytes, tc_module** out) { *out = (tc_module*)1; return 0; }
int tc_plan_create(tc_ctx* ctx, tc_plan** out) { *out = (tc_plan*)1; return 0; }
int tc_plan_free(tc_plan* p) { return 0; }
int tc_plan_add_launch(tc_plan* p, tc_module* m, const char* kernel, const uint32_t g[3], const uint32_t b[3], uint32_t smem,
                       const tc_args* args) {
  snprintf(names[calls], sizeof names[calls], "%s", kernel);
  ctrl[calls++] = (uint64_t)args->p[15];
  return 0;
}
int tc_plan_add_launch_tma(tc_plan* p, tc_module* m, const char* kernel, const uint32_t g[3], const uint32_t b[3],
                           uint32_t smem, int n, const uint64_t* desc, const tc_args* args) {
  return tc_plan_add_launch(p, m, kernel, g, b, smem, args);
}

int main(int argc, char** argv) {
  static char js[1 << 20];
  FILE* f = fopen(argv[1], "rb");
  if (argc < 3 || !f) return 2;
  js[fread(js, 1, sizeof js - 1, f)] = 0;
  fclose(f);
  int32_t keep[64];
  int n = 0;
  for (char* t = strtok(argv[2], ","); t; t = strtok(NULL, ",")) keep[n++] = atoi(t);
  tc_lowered* low = NULL;
  tc_program* prog = NULL;
  if (tc_lower_json(js, "{\"matmul\": \"tiled\"}", &low) || tc_program_create((tc_ctx*)1, low, keep, n, NULL, 0, 0, &prog)) {
    fprintf(stderr, "%s\n", tc_last_error());
    return 3;
  }
  /* the last buffer cleared while the program was made is the control blocks' */
  const uint64_t base = last_clear.p, bytes = last_clear.bytes;
  for (int k = 0; k < calls; ++k)
    printf("call %s %lld\n", names[k], ctrl[k] >= base && ctrl[k] < base + bytes ? (long long)(ctrl[k] - base) : -1LL);
  memset((void*)base, 1, bytes);
  const int status = tc_program_check(prog);
  uint64_t left = 0;
  for (uint64_t i = 0; i < bytes / 4; ++i) left += ((uint32_t*)base)[i] != 0;
  printf("check %d left %llu of %llu again %d\n", status, (unsigned long long)left, (unsigned long long)(bytes / 4), tc_program_check(prog));
  tc_program_free(prog);
  tc_lowered_free(low);
  return 0;
}
