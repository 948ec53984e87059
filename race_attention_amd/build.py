"""Build the gfx950 HIP library race_attention_amd/librace_attention.so and the
autograd calls over it, race_attention_amd/_race_torch.so.

The library is two translation units compiled side by side with hipcc for gfx950
only: csrc/race_capi.hip (the attention operators; it includes their kernel sources)
and csrc/layers_capi.hip (the operators around them, likewise).  Packed-fp32 instruction
selection is disabled (-packed-fp32-ops) for all device code.  The autograd
calls (csrc/race_torch.cpp, csrc/layers_torch.cpp) are host code against torch's C++ API.
"""
import os
import subprocess
import sys
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
SRCS = [os.path.join(HERE, "csrc", name) for name in ("race_capi.hip", "layers_capi.hip")]
OUT = os.path.join(HERE, "librace_attention.so")
TORCH_SRCS = [os.path.join(HERE, "csrc", name) for name in ("race_torch.cpp", "layers_torch.cpp")]
TORCH_OUT = os.path.join(HERE, "_race_torch.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-shared", "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function", "-Wno-unused-variable",
]


# host-side sanitizer build (device code unchanged): -fsanitize applies to the
# host compilation only, through -Xarch_host
SAN_OUT = os.path.join(HERE, "_san", "librace_attention_asan.so")
SAN_FLAGS = ["-g", "-fno-omit-frame-pointer", "-Xarch_host", "-fsanitize=address",
             "-Xarch_host", "-fsanitize=undefined"]


def _torch_cmd(out: str):
    import torch
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], "/opt/rocm/include"]
    return (["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-DUSE_ROCM", "-D__HIP_PLATFORM_AMD__=1",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"] + ["-I" + i for i in inc] +
            TORCH_SRCS + ["-o", out, "-L" + os.path.join(root, "lib")] +
            ["-l" + x for x in ("torch", "torch_cpu", "torch_hip", "c10", "c10_hip", "torch_python")])


def build(verbose: bool = True, sanitize: bool = False) -> str:
    """Both libraries (sanitize: the operator library alone), built side by side."""
    out = SAN_OUT if sanitize else OUT
    host = None
    if not sanitize:
        host = subprocess.Popen(_torch_cmd(TORCH_OUT + ".tmp"), stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                                text=True)
    if sanitize:
        os.makedirs(os.path.dirname(out), exist_ok=True)
    flags = FLAGS + (SAN_FLAGS if sanitize else [])
    compile_flags = [f for f in flags if f != "-shared"]
    with tempfile.TemporaryDirectory() as tmp:
        objs = [os.path.join(tmp, os.path.basename(src) + ".o") for src in SRCS]
        cmds = [[HIPCC] + compile_flags + ["-c", src, "-o", obj] for src, obj in zip(SRCS, objs)]
        link = [HIPCC] + flags + objs + ["-o", out + ".tmp"]
        if verbose:
            for cmd in cmds + [link]:
                print("build:", " ".join(cmd), flush=True)
        # compiler output to files: the processes run side by side, and a full pipe would stop one
        logs = [open(obj + ".log", "w+") for obj in objs]
        procs = [subprocess.Popen(cmd, stdout=log, stderr=subprocess.STDOUT) for cmd, log in zip(cmds, logs)]
        rc = max([abs(p.wait()) for p in procs])
        text = ""
        for log in logs:
            log.seek(0)
            text += log.read()
            log.close()
        if rc == 0:
            proc = subprocess.run(link, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
            rc, text = proc.returncode, text + proc.stdout
    if rc != 0 and host is not None:
        host.kill()
        host.wait()
    msgs = [ln for ln in text.splitlines() if "packed-fp32-ops" not in ln]
    if rc != 0:
        print("\n".join(msgs), file=sys.stderr)
        raise RuntimeError("hipcc failed building librace_attention.so")
    if verbose and msgs:
        print("\n".join(msgs))
    os.replace(out + ".tmp", out)
    if host is not None:
        text = host.communicate()[0]
        if host.returncode != 0:
            print(text, file=sys.stderr)
            raise RuntimeError("g++ failed building _race_torch.so")
        os.replace(TORCH_OUT + ".tmp", TORCH_OUT)
    return out


if __name__ == "__main__":
    build(sanitize="--sanitize" in sys.argv)
