"""Stub builds of the C ABI library, of chosen functions that do nothing, for a process of their own."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(tmp_path, names, code):
    """`code` in a process that loads a library with `names` alone."""
    src, lib = tmp_path / f'stub{len(names)}.c', tmp_path / f'stub{len(names)}.so'
    src.write_text(''.join(f'long long {n}(void) {{ return 0; }}\n' for n in names))
    subprocess.run(['gcc', '-shared', '-fPIC', '-o', str(lib), str(src)], check=True)
    return subprocess.run([sys.executable, '-c', code], cwd=ROOT, env=dict(os.environ, YOCO_Z1_LIB=str(lib)), capture_output=True,
                          text=True)
