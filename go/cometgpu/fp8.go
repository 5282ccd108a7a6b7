package cometgpu

/*
#include "comet_gpu.h"
*/
import "C"

import (
	"fmt"
	"runtime"
	"sync"
)

// Fp8Rows is a store of rows in 8-bit floating point: `capacity` slots of `dim` numbers, quantised as they are written (e4m3 codes, a power-of-two
// scale per block of 128 numbers: 1.02 bytes a number at 768 numbers a row, more where the last block is not full: 1.3 at 300, 2.1 at 64, 8.5 at 16),
// searched by inner product and read back. No training; any slot can be rewritten at any time.
// Scores are those of the quantised numbers, where the indexes of this package return the reference's exact ones: a store for candidates that are
// rescored, or for a language model that reads the best documents of a query with their probabilities.
type Fp8Rows struct {
	mu       sync.RWMutex
	h        *C.comet_fp8_rows
	ctx      *Context // keeps the context alive
	capacity int64
	dim      int
}

// Fp8Hit is one slot of a search: log softmax(scale * score) over the searched slots.
type Fp8Hit struct {
	Slot    int64
	LogProb float32
}

// Fp8Result is a query's best slots, best first, with log sum exp(scale * score) over all searched slots and the distribution's entropy (in nats).
type Fp8Result struct {
	Hits    []Fp8Hit
	LogSum  float32
	Entropy float32
}

// NewFp8Rows allocates the store; every slot holds zeros.
func NewFp8Rows(ctx *Context, capacity int64, dim int) (*Fp8Rows, error) {
	if dim <= 0 || dim > 1<<20 {
		return nil, fmt.Errorf("dimension must be positive and at most 2^20")
	}
	r := &Fp8Rows{ctx: ctx, capacity: capacity, dim: dim}
	if rc := C.comet_fp8_create(ctx.h, C.int64_t(capacity), C.int32_t(dim), &r.h); rc != C.COMET_OK {
		return nil, lastError(rc)
	}
	runtime.SetFinalizer(r, func(r *Fp8Rows) { r.Close() })
	return r, nil
}

// Close releases the device memory. The store must be closed before its Context.
func (r *Fp8Rows) Close() {
	r.mu.Lock()
	defer r.mu.Unlock()
	if r.h != nil {
		C.comet_fp8_destroy(r.h)
		r.h = nil
	}
}

// Capacity is the number of slots.
func (r *Fp8Rows) Capacity() int64 { return r.capacity }

// Dimensions is the length of a row.
func (r *Fp8Rows) Dimensions() int { return r.dim }

// Write puts vectors[i] into slots[i]; of vectors with one slot the last stays.
func (r *Fp8Rows) Write(slots []int64, vectors [][]float32) error {
	if len(slots) != len(vectors) {
		return fmt.Errorf("%d vectors and %d slots", len(vectors), len(slots))
	}
	if len(slots) == 0 {
		return nil
	}
	flat, err := r.flatten(vectors)
	if err != nil {
		return err
	}
	r.mu.Lock()
	defer r.mu.Unlock()
	if rc := C.comet_fp8_write(r.h, (*C.int64_t)(&slots[0]), (*C.float)(&flat[0]), C.int64_t(len(slots))); rc != C.COMET_OK {
		return lastError(rc)
	}
	return nil
}

// Read returns the numbers that the given slots hold.
func (r *Fp8Rows) Read(slots []int64) ([][]float32, error) {
	if len(slots) == 0 {
		return nil, nil
	}
	flat := make([]float32, len(slots)*r.dim)
	r.mu.RLock()
	rc := C.comet_fp8_read(r.h, (*C.int64_t)(&slots[0]), C.int64_t(len(slots)), (*C.float)(&flat[0]))
	r.mu.RUnlock()
	if rc != C.COMET_OK {
		return nil, lastError(rc)
	}
	out := make([][]float32, len(slots))
	for i := range out {
		out[i] = flat[i*r.dim : (i+1)*r.dim : (i+1)*r.dim]
	}
	return out, nil
}

// Search scores each query against the slots [first, first + n) and returns its k (at most 128) slots of largest scale * score as a distribution over all n.
// Every slot of the window counts: one that was never written is a row of zeros with score 0, and a row that holds a NaN makes the statistics of every query NaN.
func (r *Fp8Rows) Search(queries [][]float32, first, n int64, k int, scale float32) ([]Fp8Result, error) {
	B := len(queries)
	if B == 0 {
		return nil, nil
	}
	if k < 0 || k > 128 {
		return nil, fmt.Errorf("k %d outside [0, 128]", k)
	}
	flat, err := r.flatten(queries)
	if err != nil {
		return nil, err
	}
	slots := make([]int64, B*k+1) // (one more: &slots[0] with k == 0)
	logprobs := make([]float32, B*k+1)
	logsum := make([]float32, B)
	entropy := make([]float32, B)
	r.mu.RLock()
	rc := C.comet_fp8_search(r.h, C.int64_t(first), C.int64_t(n), (*C.float)(&flat[0]), C.int32_t(B), C.float(scale), C.int32_t(k), (*C.int64_t)(&slots[0]),
		(*C.float)(&logprobs[0]), (*C.float)(&logsum[0]), (*C.float)(&entropy[0]))
	r.mu.RUnlock()
	if rc != C.COMET_OK {
		return nil, lastError(rc)
	}
	out := make([]Fp8Result, B)
	for b := range out {
		hits := make([]Fp8Hit, 0, k)
		for i := b * k; i < (b+1)*k && slots[i] >= 0; i++ {
			hits = append(hits, Fp8Hit{Slot: slots[i], LogProb: logprobs[i]})
		}
		out[b] = Fp8Result{Hits: hits, LogSum: logsum[b], Entropy: entropy[b]}
	}
	return out, nil
}

func (r *Fp8Rows) flatten(vectors [][]float32) ([]float32, error) {
	flat := make([]float32, 0, len(vectors)*r.dim)
	for i, v := range vectors {
		if len(v) != r.dim {
			return nil, fmt.Errorf("vector %d: dimension mismatch: expected %d, got %d", i, r.dim, len(v))
		}
		flat = append(flat, v...)
	}
	return flat, nil
}
