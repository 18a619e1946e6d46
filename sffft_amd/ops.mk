# Builds libsffft_ops.so, the sequence-mixing operators beside the convolution (linear attention,
# rotary positions, block norms), a library of its own: the convolution's recipe, and so the stamp of its
# profile summaries, does not depend on it.
#   make -C sffft_amd -f ops.mk
ROCM ?= /opt/rocm
HIPCC ?= $(ROCM)/bin/hipcc
ARCH ?= gfx950
# the kernel build's flags (Makefile)
HIPFLAGS ?= -O3 -std=c++17 -fPIC --offload-arch=$(ARCH) -Xclang -target-feature -Xclang -packed-fp32-ops \
	-fno-slp-vectorize -mllvm -amdgpu-mfma-vgpr-form
OPS_HDRS := csrc/opsio.hpp csrc/ops_status.hpp ../include/sffft_ops.h ../include/sffft.h

.PHONY: all clean
all: libsffft_ops.so

_build/linattn.o: csrc/linattn.hpp
_build/ops_api.o: csrc/rotary.hpp csrc/blocknorm.hpp

# the compiler's resource report of each kernel is kept beside its object, as the kernel build does
_build/linattn.o _build/ops_api.o: _build/%.o: csrc/%.hip $(OPS_HDRS)
	@mkdir -p _build
	$(HIPCC) $(HIPFLAGS) -Rpass-analysis=kernel-resource-usage -c $< -o $@ 2> $@.resources; rc=$$?; \
	  grep -v 'remark: \|^ *[0-9]* | \|^ *| \|^In file included' $@.resources >&2; exit $$rc

libsffft_ops.so: _build/linattn.o _build/ops_api.o
	$(HIPCC) -shared --offload-arch=$(ARCH) -o $@ $^

clean:
	rm -f _build/linattn.o* _build/ops_api.o* libsffft_ops.so
