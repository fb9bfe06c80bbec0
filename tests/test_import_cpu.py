"""CPU: the package imports on a torch build without GPU support; only a call asks for it."""
import subprocess
import sys


def test_import_without_gpu_support_in_torch():
    code = ("import torch\n"
            "for name in [n for n in dir(torch._C) if n.startswith('_cuda_getCurrent')]:\n"
            "    delattr(torch._C, name)\n"
            "import nncf_amd\n"
            "try:\n"
            "    nncf_amd.compressed_linear(torch.zeros(2, 64, dtype=torch.float16), torch.zeros(1), None)\n"
            "except nncf_amd.errors.UnsupportedBackendError:\n"
            "    print('refused')\n")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "refused", out.stderr[-2000:]
