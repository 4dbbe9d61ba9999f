"""Two host threads, each with a context and a stream of its own, which is how the library is used from
several threads: a call of one must not change what the other's launch is allowed. The threads are C ones,
whose calls meet; Python's take turns."""
import ctypes
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CALLS = 20000  # of each thread

SOURCE = """
#include <pthread.h>
#include <string.h>
#include "zealot_attn.h"

typedef struct {
  zl_ctx* ctx;
  void *stream, *a, *b, *c, *d, *e, *f;  /* device buffers */
  int n, rows, calls, op;
  int status;
  char words[200];
} Thread;

static zl_status once(const Thread* t) {
  if (t->op == 0)  /* n tokens of one head of 256: q, positions, frequencies -> q_out */
    return zl_qk_norm_rope(t->ctx, t->a, 0, 0, 256, 0, 0, 0, 0, 1e-6f, t->b, t->c, 256, 0, t->d, 0, 0, 0, 0, 0, 0, 0, t->n, 1, 1, 256, ZL_BF16, t->stream);
  /* n requests without tokens: tables, rows, lengths -> tables, offsets, and lengths with last rows behind them */
  return zl_step_tables(t->ctx, t->a, t->rows, t->b, t->c, t->c, 0, 0, t->d, t->e, t->f, 0, 0, (int32_t*)t->f + t->n, t->n, 0, 1, 16, 1, t->stream);
}
static void* loop(void* p) {
  Thread* t = p;
  for (int i = 0; i < t->calls && t->status == 0; i++)
    if ((t->status = once(t)) != 0) strncpy(t->words, zl_last_error(), sizeof t->words - 1);
  return 0;
}
int both(Thread* t) {
  pthread_t other;
  if (pthread_create(&other, 0, loop, t + 1)) return -1;
  loop(t);
  return pthread_join(other, 0);
}
"""


class Thread(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("ctx", "stream", "a", "b", "c", "d", "e", "f")] + [
        (n, ctypes.c_int) for n in ("n", "rows", "calls", "op", "status")] + [("words", ctypes.c_char * 200)]


@pytest.fixture(scope="module")
def both(tmp_path_factory):
    d = tmp_path_factory.mktemp("threads")
    (d / "threads.c").write_text(SOURCE)
    lib = os.path.join(ROOT, "zealot_b200")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-pthread", "-I", os.path.join(ROOT, "include"), str(d / "threads.c"),
                    "-o", str(d / "threads.so"), f"-L{lib}", "-l:libzealot_attn.so", f"-Wl,-rpath,{lib}"], check=True)
    return ctypes.CDLL(str(d / "threads.so")).both


def run(both, op, sizes, buffers):
    import torch
    import zealot_b200 as zb
    ctxs, streams = [zb.GpuContext(0) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    keep = [buffers(*s) for s in sizes]
    threads = (Thread * 2)(*(Thread(c.address, s.cuda_stream, *(t.data_ptr() for t in b), **dict(zip("abcdef"[len(b):], [None] * 6)),
                                    n=n, rows=rows, calls=CALLS, op=op)
                             for c, s, b, (n, rows) in zip(ctxs, streams, keep, sizes)))
    torch.cuda.synchronize()
    assert both(threads) == 0
    torch.cuda.synchronize()
    for t, c in zip(threads, ctxs):
        assert t.status == 0, t.words
        c.check_status()
        c.close()


def test_rotation_of_many_and_of_fewer_tokens(ctx, both):
    """9,472 tokens are 16 to a CTA, 1,300 are 3: 48 KB of shared memory for copies and angles, and 35."""
    import torch
    new = lambda *s, dtype: torch.zeros(s, dtype=dtype, device="cuda")
    run(both, 0, ((9472, 0), (1300, 0)), lambda n, _: (
        new(n, 256, dtype=torch.bfloat16), new(n, dtype=torch.int32), new(128, dtype=torch.float64), new(n, 256, dtype=torch.bfloat16)))


def test_step_tables_of_many_and_of_fewer_requests(ctx, both):
    """8,192 requests with 2^18 table rows, and 2,100 with as many: 192 KB of shared memory, and 34."""
    import torch
    new = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
    run(both, 1, ((8192, 1 << 18), (2100, 2100)), lambda n, rows: (
        new(rows, 1), torch.arange(n, dtype=torch.int32, device="cuda"), new(n), new(n), new(n + 1), new(2 * n)))
