"""A double of the device library for tests of the host runtime without a GPU.

Every function of include/pt_hip.h that the operators' plans reach is there: memory lives on the host and starts as
NaN, kernels compute nothing, and the operators with several results write one value of their own into each of them, so
that a result which no call has written shows.  Calls are counted by name, and what a capture records (events, waits,
launches, with their streams) is kept as text.  A script runs in a process of its own, against a copy of the host
runtime beside the double."""
import os
import re
import shutil
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOST = os.path.join(ROOT, "php-gpu-tensors_amd", "lib", "libphptensors_host.so")

HEAD = r"""
#include "pt_hip.h"
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
static struct { const char *name; long n; } counts[256];
static long tally(const char *name, long add)
{
    int i = 0;
    while (counts[i].name && strcmp(counts[i].name, name)) i++;
    counts[i].name = name;
    return counts[i].n += add;
}
long double_count(const char *name) { return tally(strdup(name), 0); }
static char text[1 << 20];
static int capturing;
static void *current;
static void say(const char *what, void *a, void *b)
{
    if (capturing) sprintf(text + strlen(text), "%s %ld %ld\n", what, (long)a, (long)b);
}
const char *double_record(void) { return text; }
static void floats(void *p, size_t n, float x) { for (size_t i = 0; p && i < n; i++) ((float *)p)[i] = x; }
static void values(void *p, size_t n, float x, int dtype)
{
    unsigned bits;
    memcpy(&bits, &x, 4);
    if (dtype == PT_FLOAT32) floats(p, n, x);
    else if (dtype == PT_FLOAT64) for (size_t i = 0; p && i < n; i++) ((double *)p)[i] = x;
    else for (size_t i = 0; p && i < n; i++)  // (small numbers, exact in 16 bits)
        ((unsigned short *)p)[i] = dtype == PT_BFLOAT16 ? bits >> 16 : (bits >> 13 & 0x3FF) | ((bits >> 23 & 0xFF) - 112) << 10;
}
static float value(const void *p, int dtype)
{
    unsigned short h;
    unsigned bits;
    float x;
    if (dtype == PT_FLOAT32) return *(const float *)p;
    memcpy(&h, p, 2);
    bits = dtype == PT_BFLOAT16 ? (unsigned)h << 16 : (unsigned)(h & 0x3FF) << 13 | ((unsigned)(h >> 10) + 112) << 23;
    memcpy(&x, &bits, 4);
    return x;
}
static size_t tokens(const pt_attention_desc *d, int keys)
{
    return keys ? (d->k_starts ? d->k_rows : d->sequences * d->keys) : d->q_starts ? d->q_rows : d->sequences * d->queries;
}
"""

# what a function does besides being counted
BODY = {
    "pt_alloc": "*ptr = malloc(bytes + 64); memset(*ptr, 0xFF, bytes + 64);",
    "pt_free": "free(ptr);",
    "pt_memcpy_h2d": "memcpy(dst, src, bytes);", "pt_memcpy_d2h": "memcpy(dst, src, bytes);",
    "pt_memcpy_d2d": "memcpy(dst, src, bytes);",
    "pt_default_stream": "return current;", "pt_stream_set_current": "current = stream;",
    "pt_runtime_is_own": "return 1;",
    "pt_stream_create": "static long n; *stream = (pt_stream_t)++n;",
    "pt_event_create": "static long n; *event = (pt_event_t)++n;",
    "pt_event_record": 'say("record", event, stream ? stream : current);',
    "pt_stream_wait_event": 'say("wait", stream, event);',
    "pt_graph_begin_capture": "capturing = 1; text[0] = 0;",
    "pt_graph_end_capture": "capturing = 0; *graph = (pt_graph_t)1;",
    "pt_graph_end_capture_update": "capturing = 0;",
    "pt_workspace_end": "if (peak_bytes) *peak_bytes = 4096;",
    "pt_launch": 'say("launch", current, 0);', "pt_matmul": 'int full = 1; for (int i = 0; i < nd_c; i++) full = full && shape_c[i]; if (full) say("launch", current, 0);',
    "pt_reduce": 'say("launch", current, 0);',
    "pt_attention": 'say("launch", current, 0);'
                    "values(out, tokens(desc, 0) * desc->heads * desc->head_size, 1.5f, desc->dtype);"
                    "values(rest, tokens(desc, 0) * desc->heads * desc->head_size, 0.5f, desc->dtype);"
                    " floats(lse, tokens(desc, 0) * desc->heads, 2.5f);",
    # (what the forward pass left is read back, so that a gradient of unwritten results shows)
    "pt_attention_backward": 'say("launch", current, 0);'
                             "const float x = value(out, desc->dtype) + *lse;"
                             "values(dq, tokens(desc, 0) * desc->heads * desc->head_size, x + 1.0f, desc->dtype);"
                             "values(dk, tokens(desc, 1) * desc->kv_heads * desc->head_size, x + 2.0f, desc->dtype);"
                             "values(dv, tokens(desc, 1) * desc->kv_heads * desc->head_size, x + 3.0f, desc->dtype);",
    "pt_layernorm_backward": 'say("launch", current, 0);'
                             "values(dinput, rows * n, 5.0f, input_dtype); values(dgamma, n, 6.0f, param_dtype); values(dbeta, n, 7.0f, param_dtype);",
    "pt_logprobs": 'say("launch", current, 0);'
                   "floats(logprob, rows, 1.5f); floats(entropy, rows, 2.5f); floats(stats, 2 * rows, 3.5f);"
                   "floats(top_logprob, rows * top, 4.5f); for (size_t i = 0; i < rows * top; i++) top_index[i] = 7;",
    "pt_logprobs_backward": 'say("launch", current, 0); values(dlogits, rows * classes, stats[1] + (entropy ? entropy[0] : 0.0f), dtype);',
}

SCRIPT = """
import sys, ctypes
sys.path.insert(0, {package!r})
from phptensors import _abi, _host
_abi.LIB_DIR, _abi.DEVICE_LIB = {folder!r}, {device!r}
_abi.load.__defaults__ = ({device!r},)
_host.HOST_LIB = {host!r}
import numpy as np
from phptensors import CudaArray, Fusion, Sequences
lib = _abi.load()
lib.double_count.restype, lib.double_record.restype = ctypes.c_long, ctypes.c_char_p
def count(name): return lib.double_count(name.encode())
def record(): return [(w, int(a), int(b)) for w, a, b in (l.split() for l in lib.double_record().decode().splitlines())]
"""


def source():
    with open(os.path.join(ROOT, "include", "pt_hip.h")) as f:
        header = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    out = [HEAD]
    for result, name, args in re.findall(r"^([a-z][\w ]*?[ *]+)(pt_\w+)\s*\(([^;{]*?)\)\s*;", header, flags=re.M | re.S):
        if "typedef" in result:
            continue
        args, result = " ".join(args.split()), result.strip()
        body = BODY.get(name, "")
        for kind in ("pt_module_t", "pt_function_t"):
            made = re.findall(kind + r" \*\s*(\w+)", args)
            if made:
                body += f"*{made[0]} = ({kind})1;"
        last = "" if result == "void" or body.startswith("return") else 'return "";' if "char" in result else "return 0;"
        out.append(f'{result} {name}({args}) {{ tally("{name}", 1); {body} {last} }}')
    return "\n".join(out)


def build(folder):
    """The double and the host runtime beside it."""
    src = os.path.join(folder, "double.c")
    with open(src, "w") as f:
        f.write(source())
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-w", "-I", os.path.join(ROOT, "include"), src, "-o",
                    os.path.join(folder, "libpt_hip.so")], check=True)
    shutil.copy(HOST, folder)


def run(folder, code):
    head = SCRIPT.format(package=os.path.join(ROOT, "php-gpu-tensors_amd"), folder=folder, device=os.path.join(folder, "libpt_hip.so"),
                         host=os.path.join(folder, "libphptensors_host.so"))
    child = subprocess.run([sys.executable, "-c", head + code], capture_output=True, text=True, timeout=120)
    assert child.returncode == 0, child.stdout[-2000:] + child.stderr[-3000:]
    return child.stdout
