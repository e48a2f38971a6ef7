# Builds the gfx950 kernel library and the C-ABI in-tree (the .so travels with the tree; it is git-ignored).
HIPCC ?= /opt/rocm/bin/hipcc
ARCH  ?= gfx950
CSRC  := multimae_amd/csrc
OBJ   := build/obj
SRCS  := $(wildcard $(CSRC)/*.hip)
OBJS  := $(patsubst $(CSRC)/%.hip,$(OBJ)/%.o,$(SRCS)) $(OBJ)/error.o $(OBJ)/comm.o
LIB   := multimae_amd/libmmae_hip.so
# Packed fp32 instructions stay off: some of their forms have given wrong results on this chip now and then.  The step costs
# the same without them (26.93 and 26.99 ms).  The host pass does not know the feature and says so.
FLAGS := --offload-arch=$(ARCH) -O3 -fPIC -std=c++17 -Wall -Wno-unused-variable -Wno-unused-but-set-variable \
         -Xclang -target-feature -Xclang -packed-fp32-ops

all: $(LIB)

$(OBJ)/%.o: $(CSRC)/%.hip $(CSRC)/common.h $(CSRC)/ln_rows.h $(CSRC)/classdist.h include/mmae.h Makefile
	@mkdir -p $(OBJ)
	$(HIPCC) $(FLAGS) -c $< -o $@

$(OBJ)/error.o: $(CSRC)/error.cpp include/mmae.h Makefile
	@mkdir -p $(OBJ)
	$(HIPCC) $(FLAGS) -c $< -o $@

$(OBJ)/comm.o: $(CSRC)/comm.cpp include/mmae.h Makefile
	@mkdir -p $(OBJ)
	$(HIPCC) $(FLAGS) -c $< -o $@

$(LIB): $(OBJS)
	$(HIPCC) --offload-arch=$(ARCH) -shared -fPIC -o $@ $(OBJS) -ldl

clean:
	rm -rf build $(LIB)
.PHONY: all clean
