/**
 * What a decoder keeps between tokens: a paged key-value cache (append, attention of one new
 * token, eviction by accumulated weight) and the state of linear attention with a decay.  The
 * pools of the cache are updated in place; every other tensor is a value.
 * Python twin (executed by the tests): tfjs_b200/kernels/decoder.py.
 */
import {KernelConfig, KernelFunc, TensorInfo} from '@tensorflow/tfjs-core';

import {CudaBackend} from '../backend_cuda';
import {binding, packLinearAttentionParams, packPagedParams} from '../binding';

type Inputs = {[k: string]: TensorInfo};
type Args = {inputs: Inputs, attrs: {[k: string]: unknown}, backend: CudaBackend};
const asFunc = (f: (a: Args) => TensorInfo|TensorInfo[]) => f as unknown as KernelFunc;

/** `shape` holds sizes, or null where any size goes. */
function want(name: string, what: string, t: TensorInfo, shape: Array<number|null>, dtype: string): void {
  if (t.dtype !== dtype || t.shape.length !== shape.length || shape.some((w, i) => w != null && w !== t.shape[i])) {
    throw new Error(`${name}: ${what} must be ${dtype} [${shape.map(w => w ?? 'any')}], but got ${t.dtype} [${t.shape}]`);
  }
  if (t.shape.some(d => d > 2 ** 31 - 1)) {
    throw new Error(`${name}: ${what} has a dimension above 2^31 - 1: [${t.shape}]`);
  }
  if (t.shape.some(d => d <= 0)) throw new Error(`${name}: ${what} has an empty dimension: [${t.shape}]`);
}

/** Checks the pools, the table and the lengths; the dimensions and the rows' capacity. */
function paged(name: string, inp: Inputs) {
  const {kCache, vCache, pageTable, lengths} = inp;
  want(name, 'kCache', kCache, [null, null, null, null], 'float32');
  want(name, 'vCache', vCache, kCache.shape, 'float32');
  if (kCache.dataId === vCache.dataId) throw new Error(`${name}: kCache and vCache are the same tensor`);
  want(name, 'lengths', lengths, [null], 'int32');
  const batch = lengths.shape[0];
  want(name, 'pageTable', pageTable, [batch, null], 'int32');
  const [numPages, kvHeads, pageSize, headDim] = kCache.shape;
  const maxPages = pageTable.shape[1];
  return {batch, kvHeads, headDim, numPages, pageSize, maxPages, capacity: maxPages * pageSize};
}

function notAPool(name: string, inp: Inputs, names: string[]): void {
  for (const n of names) {
    const id = inp[n]?.dataId;
    if (id != null && (id === inp['kCache'].dataId || id === inp['vCache'].dataId)) {
      throw new Error(`${name}: ${n} is one of the pools`);
    }
  }
}

/** Allocates the outputs, makes the call with their device ids, and gives them back. */
function outputs(backend: CudaBackend, shapes: Array<[number[], 'float32'|'int32']>,
                 call: (ids: number[]) => void): TensorInfo[] {
  const outs: TensorInfo[] = [];
  try {
    for (const [shape, dtype] of shapes) outs.push(backend.makeOutput(shape, dtype));
    call(outs.map(o => backend.deviceId(o)));
  } catch (e) {
    outs.forEach(o => backend.disposeData(o.dataId));
    throw e;
  }
  return outs;
}

const fround = (x: unknown) => x != null ? Math.fround(x as number) : null;

export const decoderConfigs: KernelConfig[] = [
  {kernelName: '_PagedCacheAppend', backendName: 'cuda', kernelFunc: asFunc(({inputs, backend}) => {
    const name = '_PagedCacheAppend';
    const d = paged(name, inputs);
    const {kCache, vCache, k, v, pageTable, lengths, counts} = inputs;
    want(name, 'k', k, [d.batch, d.kvHeads, null, d.headDim], 'float32');
    want(name, 'v', v, k.shape, 'float32');
    if (counts != null) want(name, 'counts', counts, [d.batch], 'int32');
    notAPool(name, inputs, ['k', 'v']);
    const reads = [k, v, pageTable, lengths, counts].map(t => backend.deviceId(t));
    const [kc, vc] = [kCache, vCache].map(t => backend.deviceIdForUpdate(t));
    return outputs(backend, [[[d.batch], 'int32']], ([out]) => binding.pagedCacheAppend(
        backend.ctx, packPagedParams({...d, tokens: k.shape[2]}), kc, vc, reads[0], reads[1], reads[2], reads[3],
        reads[4], out))[0];
  })},
  {kernelName: '_PagedAttention', backendName: 'cuda', kernelFunc: asFunc(({inputs, attrs, backend}) => {
    const name = '_PagedAttention';
    const d = paged(name, inputs);
    const {q, kCache, vCache, pageTable, lengths, mask, weights} = inputs;
    want(name, 'q', q, [d.batch, null, 1, d.headDim], 'float32');
    const heads = q.shape[1];
    if (heads % d.kvHeads !== 0) {
      throw new Error(`${name}: ${heads} query heads do not share ${d.kvHeads} key-value heads evenly`);
    }
    if (mask != null) want(name, 'mask', mask, [d.batch, d.capacity], 'float32');
    if (weights != null) want(name, 'weights', weights, [d.batch, d.kvHeads, d.capacity], 'float32');
    const ids = [q, kCache, vCache, pageTable, lengths, mask, weights].map(t => backend.deviceId(t));
    const shapes: Array<[number[], 'float32'|'int32']> = [[[d.batch, 1, heads, d.headDim], 'float32']];
    if (weights != null) shapes.push([weights.shape, 'float32']);
    const outs = outputs(backend, shapes, out => binding.pagedAttention(
        backend.ctx, packPagedParams({...d, heads}, fround(attrs['scale'])), ids[0], ids[1], ids[2], ids[3], ids[4],
        ids[5], ids[6], out[0], out[1] ?? 0));
    return weights != null ? outs : outs[0];
  })},
  {kernelName: '_PagedCacheEvict', backendName: 'cuda', kernelFunc: asFunc(({inputs, attrs, backend}) => {
    const name = '_PagedCacheEvict';
    const d = paged(name, inputs);
    const {kCache, vCache, weights, pageTable, lengths, positions, total} = inputs;
    const slots = [d.batch, d.kvHeads, d.capacity];
    want(name, 'weights', weights, slots, 'float32');
    if (positions != null) want(name, 'positions', positions, slots, 'int32');
    if (total != null) want(name, 'total', total, [d.batch], 'int32');
    notAPool(name, inputs, ['weights']);
    const budget = attrs['budget'] as number, recent = (attrs['recent'] as number) ?? 0;
    if (!(budget > 0 && budget < 2 ** 30 && recent >= 0 && recent <= budget && Number.isInteger(budget) &&
          Number.isInteger(recent))) {
      throw new Error(`${name}: the budget must be a positive whole number and hold the recent slots, ` +
                      `but got budget ${budget}, recent ${recent}`);
    }
    const reads = [weights, pageTable, lengths, positions, total].map(t => backend.deviceId(t));
    const [kc, vc] = [kCache, vCache].map(t => backend.deviceIdForUpdate(t));
    return outputs(backend, [[slots, 'float32'], [slots, 'int32'], [[d.batch], 'int32'],
                             [[d.batch, d.kvHeads, budget], 'int32']],
                   out => binding.pagedCacheEvict(
                       backend.ctx, packPagedParams({...d, budget, recent}), kc, vc, reads[0], reads[1], reads[2],
                       reads[3], reads[4], out[0], out[1], out[2], out[3]));
  })},
  {kernelName: '_LinearAttention', backendName: 'cuda', kernelFunc: asFunc(({inputs, attrs, backend}) => {
    const name = '_LinearAttention';
    const {q, k, v, logDecay, state, lengths} = inputs;
    want(name, 'q', q, [null, null, null, null], 'float32');
    const [batch, heads, seq, dimK] = q.shape;
    want(name, 'k', k, q.shape, 'float32');
    want(name, 'v', v, [batch, heads, seq, null], 'float32');
    const dimV = v.shape[3];
    want(name, 'logDecay', logDecay, [heads], 'float32');
    const states = [batch, heads, dimK, dimV];
    if (state != null) want(name, 'state', state, states, 'float32');
    if (lengths != null) want(name, 'lengths', lengths, [batch], 'int32');
    const ids = [q, k, v, logDecay, state, lengths].map(t => backend.deviceId(t));
    return outputs(backend, [[[batch, seq, heads, dimV], 'float32'], [states, 'float32']],
                   out => binding.linearAttention(
                       backend.ctx, packLinearAttentionParams(batch, heads, seq, dimK, dimV, fround(attrs['scale'])),
                       ids[0], ids[1], ids[2], ids[3], ids[4], ids[5], out[0], out[1]));
  })},
];
