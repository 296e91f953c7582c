/**
 * generate(mode "sample") of HipPetitGPT beside its other modes.
 *   node run_sample_modes.mjs <model.pgw> <spec.json>   -> prints one JSON line
 * spec: { prompt: [...], maxNewTokens, temperature, numbers: [...] }
 * `kept`: the class's logits buffer is what it was before the call.
 */
import fs from "fs";
import { parsePgw } from "../../microllm-lab_amd/js/weights.mjs";
import { HipPetitGPT } from "../../microllm-lab_amd/js/engine.mjs";

async function main() {
  const [, , pgwPath, specPath] = process.argv;
  const spec = JSON.parse(fs.readFileSync(specPath, "utf8"));
  const model = new HipPetitGPT(parsePgw(fs.readFileSync(pgwPath)));
  let at = 0;
  model._logits.fill(7);
  const drawn = await model.generate(spec.prompt, Object.assign({}, spec, {
    mode: "sample",
    random: () => spec.numbers[at++],
  }));
  const kept = model._logits.every((v) => v === 7);
  const greedy = await model.generate(spec.prompt, { maxNewTokens: spec.maxNewTokens });
  model.destroy();
  console.log(JSON.stringify({ drawn: drawn.generatedIds, kept, greedy: greedy.generatedIds }));
}

main().catch((e) => {
  console.error(e && e.stack ? e.stack : String(e));
  process.exit(1);
});
