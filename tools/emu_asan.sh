#!/bin/bash
# CPU container: the kernel sources on the fiber emulator, every translation unit of the library, built with host
# AddressSanitizer and with every workgroup's LDS poisoned (tests/emu/hip_emu.h: poison_lds), through the emulator parity tests
# and the checks of the language-model operators: the sanitizer pass of the device code.
#   bash tools/emu_asan.sh [pytest -k expression]      -> build/emu_asan.log
set -u
cd "$(dirname "$0")/.."
mkdir -p build
LIB="$(python -c "import __graft_entry__ as ge; print(ge.build_emu_variant('asan', ['-fsanitize=address', '-fno-omit-frame-pointer']))")" || exit 1
K="${1:-not cli and not host and not train}"
LD_PRELOAD="$(gcc -print-file-name=libasan.so)" ASAN_OPTIONS=detect_leaks=0 JPPEMU_TEST_LIB="$LIB" \
  timeout 3000 python -m pytest tests/test_cpu_parity.py tests/test_ref_fixtures.py tests/test_scorers.py tests/test_lm_cpu.py -x -q -m "not gpu" -k "$K" > build/emu_asan.log 2>&1
echo "rc $?"; grep -v "^  File" build/emu_asan.log | tail -15
